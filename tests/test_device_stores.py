"""How device code may write: through vector stores only.

The scalar data cache is not kept coherent with the vector caches: a kernel that wrote through it would have to write the cache back by hand before anyone else may read the data.
So no source here holds a scalar store, a scalar atomic or that cache's write-back or discard."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = (".hip", ".h", ".hpp", ".c", ".cpp", ".s", ".py", ".sh")
# (in pieces: this file is among those searched)
SCALAR_WRITE = re.compile(r"s_(?:buffer_|scratch_)?" r"sto" r"re|s_(?:buffer_)?" r"ato" r"mic|s_dcache_" r"(?:wb|discard)")


def _sources():
    for top in ("falcon_unzip_amd", "include", "oracle", "scripts", "tests", "tools"):
        for d, _, names in os.walk(os.path.join(ROOT, top)):
            for n in names:
                if n.endswith(CODE) or n == "Makefile":
                    yield os.path.join(d, n)
    for n in ("bench.py", "__graft_entry__.py"):
        yield os.path.join(ROOT, n)


def test_the_pattern_knows_the_instructions():
    st, at = "sto" + "re", "ato" + "mic"
    for ins in ("s_%s_dwordx4" % st, "s_buffer_%s_dword" % st, "s_scratch_%s_dword" % st, "s_%s_add" % at, "s_buffer_%s_swap" % at, "s_dcache_" + "wb", "s_dcache_" + "wb_vol", "s_dcache_" + "discard"):
        assert SCALAR_WRITE.search(ins), ins
    for ins in ("s_load_dwordx4", "s_dcache_inv", "global_" + st + "_dwordx4", "buffer_" + st + "_dword", "global_" + at + "_add"):
        assert not SCALAR_WRITE.search(ins), ins


def test_no_source_writes_through_the_scalar_data_cache():
    seen, bad = 0, []
    for p in _sources():
        seen += 1
        with open(p, encoding="utf-8", errors="replace") as f:
            bad += ["%s:%d" % (os.path.relpath(p, ROOT), i) for i, line in enumerate(f, 1) if SCALAR_WRITE.search(line)]
    assert seen > 60, seen
    assert not bad, bad
