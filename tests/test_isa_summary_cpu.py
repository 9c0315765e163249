"""scripts/isa_summary.py describes the kernels of libgvk.so as they are built: every file of them, with the Makefile's flags."""
import importlib.util
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "graphvite_amd", "csrc")


def test_it_takes_the_makefile_s_sources_and_flags():
    spec = importlib.util.spec_from_file_location("isa_summary", os.path.join(ROOT, "scripts", "isa_summary.py"))
    summary = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(summary)
    # make, asked what it would do for an empty tree
    dry = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout
    compiled = [line.split() for line in dry.splitlines() if " -c " in line and ".hip " in line]
    assert compiled and sorted(os.path.basename(words[words.index("-c") + 1]) for words in compiled) == summary.sources()
    assert "gvk_blocks.hip" in summary.sources() and "gvk_logits.hip" in summary.sources()
    for words in compiled:
        built = [os.path.normpath(w) if w.startswith("-I") else w for w in words[1:words.index("-c")]]
        assert built == [os.path.normpath(w) if w.startswith("-I") else w for w in summary.flags()]
    assert "-packed-fp32-ops" in summary.flags()
