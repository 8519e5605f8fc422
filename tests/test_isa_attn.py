"""The built attention kernels' direct-to-LDS loads: none is in flight at a barrier that publishes its tile, and the next tile's
stay in flight over this one's products (a wait for them in front of the fragment reads would serialise the two)."""
from __future__ import annotations

from tests.test_isa_waits import _lds_dma, _successors, _vmcnt, kernels  # noqa: F401


def _direct(kernels):  # noqa: F811
    return {n: c for n, c in kernels.items() if ("attn_tile_kernel" in n or "attn_mixed_kernel" in n) and any(_lds_dma(m, o) for _, m, o in c)}


def _walk(code, start, stop):
    """Indices at which the paths from code[start] end: stop(i) says "end" or "cut"."""
    addr = {a: i for i, (a, _, _) in enumerate(code)}
    ends, seen, todo = set(), set(), _successors(code, addr, start)
    while todo:
        i = todo.pop()
        if i in seen:
            continue
        seen.add(i)
        what = stop(i)
        if what == "end":
            ends.add(i)
        elif what is None:
            todo += _successors(code, addr, i)
    return ends


def test_tiles_have_landed_at_their_barrier(kernels):  # noqa: F811
    found = _direct(kernels)
    assert len(found) == 12, sorted(found)  # two types, three head sizes, alone and among items of few rows
    for name, code in found.items():
        for k, (_, m, o) in enumerate(code):
            if _lds_dma(m, o):
                ends = _walk(code, k, lambda i: "cut" if _vmcnt(code[i][1], code[i][2]) == 0 else (
                    "end" if code[i][1] in ("s_barrier", "s_endpgm") else None))
                assert not ends, f"{name}: the load at {k} may be in flight at {ends}"


def test_the_next_tile_is_loaded_over_the_products(kernels):  # noqa: F811
    for name, code in _direct(kernels).items():
        over = [k for k, (_, m, o) in enumerate(code) if _lds_dma(m, o) and _walk(
            code, k, lambda i: "cut" if _vmcnt(code[i][1], code[i][2]) is not None else ("end" if "mfma" in code[i][1] else None))]
        assert len(over) >= 8, (name, over)
