"""The plan refuses outputs that overlap what its blocks of threads read, or each other.  Every
block scans all lengths while the first one writes ``seq_lens``, so lengths updated in place would
race from the second block on; the refusal comes before any CUDA call.  CPU only."""
from __future__ import annotations

import pytest

from triton_fused_rmsnorm_qkv import _lib

A = 1 << 32  # fake addresses far apart, never dereferenced
R, T, WIDTH, STRIDE, CAP = 5, 4000, 7, 9, 50
SIZES = dict(ctx=R, new=R, free=CAP, n_free=1, start=R + 1, positions=T, slots=T, lens=R, n_free_out=1, refused=1)
READ, WRITTEN = ("ctx", "new", "free", "n_free"), ("start", "positions", "slots", "lens", "n_free_out", "refused")


def plan(**kw):
    a = dict(ctx=A, new=2 * A, R=R, table=3 * A, stride=STRIDE, width=WIDTH, free=4 * A, cap=CAP, n_free=5 * A, block=16,
             T=T, start=6 * A, positions=7 * A, slots=8 * A, lens=9 * A, n_free_out=10 * A, refused=11 * A, flags=8,
             stream=None)  # flags 8 is refused after the overlaps, so that nothing is ever launched
    a.update(kw)
    _lib.load()
    return _lib.kv4["plan"](*a.values())


def place(name):
    return dict(ctx=A, new=2 * A, free=4 * A, n_free=5 * A, start=6 * A, positions=7 * A, slots=8 * A, lens=9 * A,
                n_free_out=10 * A, refused=11 * A)[name]


@pytest.mark.parametrize("out", WRITTEN)
@pytest.mark.parametrize("other", READ + WRITTEN)
def test_plan_refuses_overlaps(out, other):
    if out == other:
        return
    at = place(other)
    for offset in {0, 4 * (SIZES[other] - 1), -4 * (SIZES[out] - 1)}:  # same start, last word, first word
        assert plan(**{out: at + offset}) == _lib.ERR_ALIAS, offset
        assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("name", READ + WRITTEN)
def test_plan_refuses_overlaps_with_the_tables(name):
    row = 4 * STRIDE
    for at in (0, 4 * (WIDTH - 1), row, 3 * row + 8, (R - 1) * row + 4 * (WIDTH - 1), -4 * (SIZES[name] - 1)):
        assert plan(**{name: 3 * A + at}) == _lib.ERR_ALIAS, at


def test_what_does_not_overlap_is_not_refused():
    """Neighbours, and a word between the rows of a strided table: past the check, to that of the flags."""
    for kw in (dict(lens=A + 4 * R), dict(lens=A - 4 * R), dict(refused=3 * A + 4 * WIDTH),
               dict(n_free_out=3 * A + 4 * (STRIDE * (R - 1) + WIDTH)), dict(new=A), dict(n_free=4 * A)):
        assert plan(**kw) == _lib.ERR_SCHEDULE, kw
