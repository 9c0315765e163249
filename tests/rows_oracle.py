"""Plain 64-bit restatements of the whole-row operators of include/gvk.h (8-bit block tables, their logits, top logits, distillation)."""
import numpy as np


def quantise(x):
    """float array [rows, dim] -> (float64 values x stands for, exponent bytes [rows, blocks]); NaN / infinity mark a block."""
    x = np.asarray(x, np.float64)
    rows, dim = x.shape
    out, exponents = np.zeros_like(x), np.zeros((rows, -(-dim // 128)), np.uint8)
    for b in range(exponents.shape[1]):
        part = x[:, 128 * b:128 * b + 128]
        bad = ~np.isfinite(part).all(1)
        largest = np.where(bad, 1.0, np.abs(np.where(np.isfinite(part), part, 0)).max(1))
        power = np.full(rows, 0, np.int64)
        for r in np.nonzero(largest > 0)[0]:
            e = int(np.floor(np.log2(largest[r]))) - 10
            while largest[r] > 448.0 * 2.0 ** e:  # the least power of two that brings the block to 448 or below
                e += 1
            power[r] = max(e, -127)
        scale = np.exp2(power.astype(np.float64))[:, None]
        y = np.where(bad[:, None], 0, part) / scale
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        y = np.rint(y / step) * step * scale
        out[:, 128 * b:128 * b + 128] = np.where(bad[:, None], np.nan, y)
        exponents[:, b] = np.where(bad, 255, np.where(largest == 0, 127, power + 127))
    return out, exponents


def top(z, k, temperature):
    """(values, index, stats) of float64 rows; NaN first, of equal logits the lowest candidate."""
    z = np.asarray(z, np.float64) + 0.0
    key = np.where(np.isnan(z), np.inf, z)
    nan = np.isnan(z)
    index = np.stack([np.lexsort((np.arange(z.shape[1]), -key[r], ~nan[r])) for r in range(len(z))])[:, :k]
    with np.errstate(all="ignore"):
        m = np.where(nan, -np.inf, z).max(1)
        base = np.where(m == -np.inf, 0, m)
        stats = np.stack([m, np.log(np.exp((z - base[:, None]) / temperature).sum(1))], 1)
    return np.take_along_axis(z, index, 1), index, stats


def distill(z, index, teacher, temperature, teacher_stats=None, weight=None):
    """(loss, stats, grad, scale of the gradient's terms, scale of the loss's terms) in float64, row by row from the formulas."""
    z = np.asarray(z, np.float64)
    rows, n = z.shape
    loss, stats, grad = np.zeros(rows), np.zeros((rows, 2)), np.zeros((rows, n))
    grad_scale, loss_scale = np.zeros((rows, n)), np.zeros(rows)
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = z[r].max()
            e = np.exp((z[r] - (0 if m == -np.inf else m)) / temperature)
            stats[r] = m, np.log(e.sum())
            entries = [(i, t) for i, t in zip(index[r].tolist(), np.asarray(teacher[r], np.float64).tolist()) if i != -1 and t != -np.inf]
            if any(i < -1 or i >= n for i in index[r]):
                loss[r], grad[r] = np.nan, np.nan
                continue
            if not entries or m == -np.inf:
                continue
            t = np.array([x[1] for x in entries])
            if teacher_stats is None:
                log_q = (t - t.max()) / temperature
                log_q = log_q - np.log(np.exp(log_q).sum())
            else:
                log_q = (t - float(teacher_stats[r][0])) / temperature - float(teacher_stats[r][1])
            q, at = np.exp(log_q), np.array([x[0] for x in entries])
            p = e / e.sum()
            log_p = (z[r] - m) / temperature - stats[r, 1]
            used = q > 0
            loss[r] = (q[used] * (log_q[used] - log_p[at[used]])).sum()
            loss_scale[r] = (q[used] * (np.abs(log_q[used]) + np.abs(log_p[at[used]]) + 1)).sum()
            listed = np.zeros(n)
            np.add.at(listed, at, q)
            w = (1.0 if weight is None else float(weight[r])) / temperature
            grad[r] = w * (q.sum() * p - listed)
            grad_scale[r] = abs(w) * (q.sum() * p + listed)
    return loss, stats, grad, grad_scale, loss_scale
