"""bench.py's arithmetic on the command line's figures."""
import importlib.util
import os

from tests.util import ROOT


def test_a_list_that_is_done_with_its_first_context_has_a_length():
    spec = importlib.util.spec_from_file_location("bench_module", os.path.join(ROOT, "bench.py"))
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    for wall, first, want in (("0.100", "0.100", 1e-3), ("0.100", "0.101", 1e-3), ("0.350", "0.100", 0.25), ("0.5", None, 0.5)):
        kv = {"wall_s": wall}
        if first:
            kv["first_ctx_s"] = first
        s = bench.list_loop_seconds(kv)
        assert abs(s - want) < 1e-9 and round(s, 3) > 0
