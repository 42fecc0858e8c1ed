"""The recorded HBM traffic of the training GEMMs is quoted by bench.py only for the sources that it was measured on: the record names their hash, and the
hash covers the GEMM headers that those sources include."""
import json
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "spatialthinker_amd", "csrc")


def test_the_hash_covers_the_gemm_headers():
    import bench
    seen, todo = set(), list(bench.GEMM_SOURCES)
    while todo:
        name = todo.pop()
        seen.add(name)
        text = open(os.path.join(CSRC, name)).read()
        todo += [h for h in re.findall(r'#include "(gemm\w*\.h)"', text) if h not in seen]
    assert seen == set(bench.GEMM_SOURCES)


def test_the_record_is_of_these_sources():
    import bench
    record = json.load(open(os.path.join(ROOT, bench.GEMM_TRAFFIC)))
    assert record["kernel_source_sha16"] == bench.gemm_source_sha()
    assert record["hbm_bytes_per_launch"] > record["algorithmic_bytes_per_launch"] > 0
