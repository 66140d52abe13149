"""The chained row filter's work tickets, read from the sources and from the compiler's output (CPU test: hipcc cross-compiles gfx950
without a GPU).

The scalar data cache is read-only to this library: whatever a kernel writes, the tickets' atomics included, goes through vector memory.
And the draw must not cost the prefetch ring: the returning atomic is requested ahead of its use, so no wait at a ticket's read inside the
loop may drain the row pairs in flight."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
CSRC = os.path.join(ROOT, "rustcv_amd", "csrc")
SCALAR_WRITE = re.compile(r"\bs_[a-z_]*(?:atomic|store|dcache)")   # (no scalar instruction that reads only is named like this)


@pytest.fixture(scope="module")
def rows_asm(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("isa") / "rows.s"
    flags = "-O3 -std=c++17 --offload-arch=gfx950 -ffp-contract=off -fno-fast-math".split()
    subprocess.check_call([HIPCC, *flags, "--cuda-device-only", "-S", "-o", str(out), os.path.join(CSRC, "rcv_filter_rows_mfma.hip")], stderr=subprocess.DEVNULL)
    return [l.split(";")[0].strip() for l in open(out)]


def test_no_source_writes_through_the_scalar_cache():
    files = [f for d, pats in ((CSRC, ("*.hip", "*.h")), (os.path.join(ROOT, "tools"), ("*.hip",)), (os.path.join(ROOT, "include"), ("*",)))
             for pat in pats for f in glob.glob(os.path.join(d, pat))]
    assert len(files) > 20
    hits = [(os.path.relpath(f, ROOT), i + 1) for f in files for i, l in enumerate(open(f, errors="replace")) if SCALAR_WRITE.search(l)]
    assert not hits, hits


def test_no_instruction_of_the_row_filter_writes_through_the_scalar_cache(rows_asm):
    hits = [l for l in rows_asm if SCALAR_WRITE.match(l)]
    assert not hits, sorted(set(hits))[:4]


@pytest.mark.parametrize("ks", [3, 5, 7])
def test_a_ticket_is_one_vector_atomic_requested_ahead(rows_asm, ks):
    i0 = next(i for i, l in enumerate(rows_asm) if re.match(r"^_Z\S*19k_filter_rows_chainILi%dELi3E\S*:" % ks, l))
    i1 = next(i for i in range(i0, len(rows_asm)) if rows_asm[i].startswith(".Lfunc_end"))
    body = [l for l in rows_asm[i0:i1] if l]
    draws = [i for i, l in enumerate(body) if "atomic" in l]
    # two queues, each: the first draw in front of the loop, the next item's at the head of a trip
    assert len(draws) == 4 and all(re.match(r"global_atomic_add_x2 v\[\d+:\d+\], .* sc0$", body[i]) for i in draws), [body[i] for i in draws]
    regs = {re.match(r"global_atomic_add_x2 v\[(\d+):", body[i]).group(1) for i in draws}
    # one lane draws: every atomic sits in a region whose exec mask was narrowed in front of it, and nothing is waited for between
    for i in draws:
        near = body[max(0, i - 10):i]
        assert any(l.startswith("s_and_saveexec_b64") or l.startswith("s_mov_b64 exec") for l in near), near
    # only the first draw of a queue waits for everything; the reads inside the loop leave at least one row pair (three loads) outstanding
    drains = 0
    reads = [i for i, l in enumerate(body) if re.match(r"v_readfirstlane_b32 s\d+, v(\d+)$", l) and l.rsplit("v", 1)[1] in regs]
    assert reads
    for i in reads:
        w = re.match(r"s_waitcnt vmcnt\((\d+)\)$", body[i - 1])
        if w and int(w.group(1)) == 0:
            drains += 1
        elif w:
            assert int(w.group(1)) >= 3, body[i - 1:i + 1]
    assert drains <= 2, drains
