"""GraphSolver.scorer / distill without a GPU: when they refuse, by the host build of the engine (tests/hostdev).  tests/test_solver_cpu.py
says how such processes run."""
import os
import sys

import pytest

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def make_solver(seed=5):
    import graphvite_amd as gv
    from graphvite_amd import synthetic
    g = gv.graph.Graph()
    g.load(synthetic.power_law_edges(250, 2500, seed=3))
    s = gv.solver.GraphSolver(32, num_sampler_per_worker=2, seed=seed)
    s.build(g, batch_size=500, episode_size=5)
    return g, s


def refused_for_a_session(s):
    """Whether scorer and distill refuse because a session is open.  They refuse here in any case: there is no GPU, and None is no teacher."""
    words = []
    for call in (s.scorer, lambda: s.distill(None)):
        with pytest.raises((RuntimeError, ValueError, TypeError)) as refusal:
            call()
        words.append("session is open" in str(refusal.value))
    assert words[0] == words[1]
    return words[0]


def sessions():
    """scorer and distill refuse while the engine has a session open, and only then: close(), train(), build(), clear() and a failed
    second session leave them as the engine says."""
    kw = dict(model="LINE", num_epoch=1, augmentation_step=1, log_frequency=100000)
    g, s = make_solver()
    assert not refused_for_a_session(s)
    session = s.session(**kw)
    assert refused_for_a_session(s)
    session.close()
    assert not refused_for_a_session(s)
    s.session(**kw)
    s.train(**kw)  # ends the session
    assert not refused_for_a_session(s) and s.predict([[0, 1]]).shape == (1,)
    s.session(**kw)
    s.build(g, batch_size=500, episode_size=5)
    assert not refused_for_a_session(s)
    s.session(**kw)
    s.clear()
    assert not refused_for_a_session(s)
    first, second = s.session(**kw), None
    with pytest.raises(ValueError):
        second = s.session(**dict(kw, model="none"))  # refused before anything is touched: the first one goes on
    assert second is None and refused_for_a_session(s)
    second = s.session(**kw)
    assert refused_for_a_session(s)
    second.close()
    assert not refused_for_a_session(s)
    with pytest.raises(ValueError, match="no open session"):
        first.close()
    assert not refused_for_a_session(s)


def _rank(rank, port):
    import torch.distributed as dist
    from graphvite_amd.scorer import LinkScorer
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK=str(rank), LOCAL_WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        _, s = make_solver()
        s.train(model="LINE", num_epoch=1, augmentation_step=1, log_frequency=100000)
        before = s.vertex_embeddings.copy(), s.context_embeddings.copy()
        with pytest.raises(ValueError, match="job of 2"):
            s.distill(LinkScorer.__new__(LinkScorer))
        assert (s.vertex_embeddings == before[0]).all() and (s.context_embeddings == before[1]).all()
    finally:
        dist.destroy_process_group()


def two_processes():
    import torch.multiprocessing as mp
    from host_scenarios import _free_port
    mp.spawn(_rank, args=(_free_port(),), nprocs=2, join=True)


@pytest.fixture(scope="module")
def run(request):
    import json
    import subprocess
    import test_solver_cpu
    root = test_solver_cpu.ROOT
    for directory in ("oracle", os.path.join("tests", "hostdev")):
        target = [os.path.join(root, "oracle", "liboracle.so")] if directory == "oracle" else []
        subprocess.check_call(["make", "-s", "-C", os.path.join(root, directory)] + target)
    env = {k: v for k, v in os.environ.items() if k not in ("RANK", "WORLD_SIZE", "LOCAL_RANK")}
    env.update(GVK_LIBRARY=test_solver_cpu.HOST_LIBRARY, GVK_ALLOW_TEST_LIBRARY="1", CUDA_VISIBLE_DEVICES="", HIP_VISIBLE_DEVICES="")

    def go(name, *arguments):
        child = subprocess.run([sys.executable, os.path.abspath(__file__), name, json.dumps(arguments)], cwd=root, env=env, capture_output=True,
                               text=True, timeout=300)
        assert child.returncode == 0, child.stdout[-3000:] + child.stderr[-6000:]
    return go


def test_a_session_s_state_is_the_engine_s(run):
    run("sessions")


def test_distill_refuses_in_a_job_of_several_processes(run):
    run("two_processes")


if __name__ == "__main__":
    import json
    import logging
    import graphvite_amd
    graphvite_amd.init_logging(logging.ERROR)
    globals()[sys.argv[1]](*json.loads(sys.argv[2]))
