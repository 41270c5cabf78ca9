"""Beam search's selection (nnb200_beam_select) against a plain 64-bit form (tests/paged_ref.py)."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    from tests import gpu_util
    return gpu_util


def _run(g, dtype, logits, scores, ended, eos, n, ld_extra=0, offset=0, with_ended_out=True):
    """logits (groups, beams, vocab) fp32 values of the type.  Returns parent, token, score, ended and checks what lies beside them."""
    import torch
    groups, beams, vocab = logits.shape
    t = torch.bfloat16 if dtype else torch.float32
    flat = torch.full((groups * beams * (vocab + ld_extra) + offset,), float("nan"), device="cuda", dtype=t)
    flat[offset:].view(groups * beams, vocab + ld_extra)[:, :vocab] = torch.from_numpy(logits.reshape(-1, vocab)).cuda()
    sc = g.dev(scores.astype(np.float32).reshape(-1))
    en = None if ended is None else g.dev(ended.astype(np.int32).reshape(-1))
    outs = [torch.full((groups * n + 2,), -9, dtype=torch.int32, device="cuda") for _ in range(3)]
    so = torch.full((groups * n + 2,), -9.0, device="cuda")
    need = g.call("nnb200_beam_select_scratch_bytes", groups, beams, vocab, n)
    scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    g.call("nnb200_beam_select", C.c_void_p(flat.data_ptr() + offset * flat.element_size()), vocab + ld_extra, dtype, groups, beams, vocab, g.ptr(sc), g.ptr(en), eos, n,
           g.ptr(outs[0]), g.ptr(outs[1]), g.ptr(so), g.ptr(outs[2]) if with_ended_out else None, g.ptr(scratch), need, g.stream())
    torch.cuda.synchronize()
    assert bool((scratch[need:] == 255).all())
    for o in outs + [so]:
        assert bool((o[groups * n:] == -9).all())
    got = [o[:groups * n].cpu().numpy().reshape(groups, n) for o in (outs[0], outs[1], so, outs[2])]
    if not with_ended_out:
        assert np.all(got[3] == -9)
    return got


def _check(g, dtype, logits, scores, ended, eos, n, **more):
    import torch
    if dtype:
        logits = torch.from_numpy(logits).bfloat16().float().numpy()
    scores = scores.astype(np.float32)
    want = ref.select(logits.astype(np.float64), scores.astype(np.float64), ended, eos, n)
    parent, token, score, out = _run(g, dtype, logits, scores, ended, eos, n, **more)
    for i, row in enumerate(want):
        assert [(int(a), int(b)) for a, b in zip(parent[i], token[i])] == [(r[0], r[1]) for r in row]
        w = np.array([r[2] for r in row])
        # one rounding to fp32, and a normaliser whose exponentials are in 32 bits: at most a few steps of 2^-23 of the sum
        with np.errstate(invalid="ignore"):
            assert np.all((np.abs(score[i] - w) <= 2.0 ** -24 * np.abs(w) + 2.0 ** -21) | (score[i] == w))
        if more.get("with_ended_out", True):
            assert [int(a) for a in out[i]] == [r[3] for r in row]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("groups,beams,vocab,n", [(1, 1, 1, 1), (1, 4, 4096, 4), (2, 1, 50, 50), (3, 8, 513, 16), (1, 64, 1000, 128), (2, 5, 33000, 10), (1, 3, 131, 128),
                                                  (5, 2, 8191, 3), (1, 2, 100003, 64), (7, 16, 2049, 32)])
def test_select(g, dtype, groups, beams, vocab, n):
    r = np.random.default_rng(groups + beams + vocab)
    logits = (3 * r.standard_normal((groups, beams, vocab))).astype(np.float32)
    scores = -np.sort(10 * r.random((groups, beams)), axis=1)
    _check(g, dtype, logits, scores, None, -1, n)
    ended = r.random((groups, beams)) < 0.4
    _check(g, dtype, logits, scores, ended, vocab // 2, n)


@pytest.mark.parametrize("dtype", [0, 1])
def test_select_ties_go_to_the_lower_beam_and_token(g, dtype):
    """Whole numbers as logits, the same in every beam: most candidates are equal to others."""
    r = np.random.default_rng(1)
    one = r.integers(0, 4, 5000).astype(np.float32)
    logits = np.stack([one, one, np.roll(one, 7), one])[None]
    _check(g, dtype, logits, np.zeros((1, 4)), None, -1, 100)
    _check(g, dtype, logits, np.array([[-1.0, 0.0, 0.0, -1.0]]), None, 3, 128)
    _check(g, dtype, np.zeros((2, 3, 20000), np.float32), np.zeros((2, 3)), None, 19999, 70)
    # logits 0 and -0 are the same number
    z = np.zeros((1, 2, 600), np.float32)
    z[:, :, ::2] = -0.0
    _check(g, dtype, z, np.zeros((1, 2)), None, -1, 40)


@pytest.mark.parametrize("dtype", [0, 1])
def test_select_sorted_rows(g, dtype):
    """The best candidates side by side, at either end of a row, in one stretch of it."""
    v = np.linspace(-8, 8, 9000, dtype=np.float32)
    _check(g, dtype, np.stack([v, v[::-1], np.roll(v, 3333)])[None].copy(), np.array([[0.0, -0.3, -0.7]]), None, -1, 128)


@pytest.mark.parametrize("dtype", [0, 1])
def test_select_masked_vocabulary(g, dtype):
    """-inf and the type's lowest value at masked tokens, whole rows of them, NaN and +inf rows, dead beams, fewer candidates than places."""
    import torch
    r = np.random.default_rng(2)
    low = float(torch.finfo(torch.bfloat16 if dtype else torch.float32).min)
    logits = (3 * r.standard_normal((6, 3, 700))).astype(np.float32)
    logits[0, :, 10:] = -np.inf
    logits[1, :, 5:] = low
    logits[2, 0], logits[2, 1, 3], logits[2, 2, 9] = -np.inf, np.nan, np.inf
    logits[3, 0], logits[3, 1, 600] = low, np.nan
    logits[5, 2, :] = np.inf
    scores = np.array([[0, -1, -2], [0, -1, -2], [0, 0, 0], [-1, -2, -3], [-np.inf, np.nan, -3], [-np.inf, -np.inf, 0]])
    _check(g, dtype, logits, scores, None, 2, 40)
    ended = np.array([[1, 0, 0], [0, 1, 1], [1, 1, 0], [0, 1, 0], [1, 0, 0], [0, 1, 1]])
    _check(g, dtype, logits, scores, ended, 2, 40)


@pytest.mark.parametrize("dtype", [0, 1])
def test_select_odd_strides_and_starts(g, dtype):
    r = np.random.default_rng(4)
    logits = (3 * r.standard_normal((2, 3, 1003))).astype(np.float32)
    for ld_extra, offset in ((5, 0), (0, 1), (1, 3), (8, 8)):
        _check(g, dtype, logits, np.zeros((2, 3)), None, 7, 12, ld_extra=ld_extra, offset=offset)


def test_select_large_and_small_logits(g):
    r = np.random.default_rng(5)
    logits = r.standard_normal((1, 4, 3001)).astype(np.float32)
    scores = -r.random((1, 4))
    _check(g, 0, logits * 1e-3, scores, None, -1, 9)
    _check(g, 0, logits * 200 + 5e4, scores, None, -1, 9)
    _check(g, 0, logits - 3e4, scores - 1e4, None, -1, 9)


def test_select_without_ended_out(g):
    logits = np.random.default_rng(6).standard_normal((2, 2, 300)).astype(np.float32)
    _check(g, 0, logits, np.zeros((2, 2)), None, 1, 5, with_ended_out=False)


def test_select_says_which_of_close_candidates_is_better(g):
    """The normaliser separates candidates a millionth apart: two beams whose scores differ by 2^-20 less what their normalisers do."""
    r = np.random.default_rng(7)
    for seed in range(20):
        base = (2 * r.standard_normal(4000)).astype(np.float32)
        other = base.copy()
        other[3000:] = (2 * r.standard_normal(1000)).astype(np.float32)
        other[3000:] = np.minimum(other[3000:], 3.0)
        x = np.stack([base, other]).astype(np.float64)
        norm = np.log(np.exp(x).sum(axis=1))
        s = np.float32(norm[1] - norm[0])
        scores = np.array([[0.0, float(s) + 2.0 ** -20 * (1 if seed % 2 else -1)]])
        _check(g, 0, x.astype(np.float32)[None], scores, None, -1, 30)


def test_select_more_candidates_than_a_tile_of_a_long_row(g):
    """Rows whose first tile of 4096 is one value and whose second lies above it but for some tokens, of which the best are spread."""
    groups, vocab, n = 600, 8192, 128
    logits = np.ones((groups, 1, vocab), dtype=np.float32)
    second = np.full((8, 128, 4), 2.0, dtype=np.float32)
    second[0, :, 0] = 3.0
    second[:, 127] = 1.0
    logits[:, 0, 4096:] = second.reshape(-1)
    _check(g, 0, logits, np.zeros((groups, 1)), None, -1, n)


def _exponential_error(v, ref_point):
    """Error of exp(v - ref_point) where v - ref_point, and its product with log2(e) in two parts, are rounded to fp32: what
    a reference point far below a logit costs."""
    d = (v - ref_point).astype(np.float32)
    hi, lo = np.float32(1.4426950216293335), np.float32(1.925963033500e-8)
    x = (d.astype(np.float64) * np.float64(hi) + (d * lo).astype(np.float64)).astype(np.float32)
    return np.exp2(x.astype(np.float64)) / np.exp(v.astype(np.float64) - ref_point.astype(np.float64)) - 1.0


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("gap", [60.0, 45.0, 25.0, 12.0, 7.0])
def test_select_rows_whose_peak_lies_far_above_their_first_tile(g, dtype, gap):
    """One logit `gap` above the first 4096, chosen so that 32 bits err upwards in one beam and downwards in the other, of
    two whose best values are 2e-6 apart; rows of two tiles that one block reads."""
    groups, vocab, half = 600, 8192, gap / 2
    r = np.random.default_rng(int(gap))
    logits = (-half - 9 + r.standard_normal((groups, 2, vocab))).clip(None, -half - 2).astype(np.float32)
    first, peak = (-half + 0.9 * r.random(400000)).astype(np.float32), (half + 0.9 * r.random(400000)).astype(np.float32)
    order = np.argsort(_exponential_error(peak, first))
    for b, picked in ((0, order[-groups:]), (1, order[:groups])):
        logits[:, b, 77], logits[np.arange(groups), b, 4096 + r.integers(0, 4096, groups)] = first[picked], peak[picked]
    if dtype:
        import torch
        logits = torch.from_numpy(logits).bfloat16().float().numpy()
    x = logits.astype(np.float64)
    top = x.max(axis=2)
    best = -np.log(np.exp(x - top[..., None]).sum(axis=2))                     # the best candidate of each beam
    scores = np.zeros((groups, 2), np.float32)
    scores[:, 1] = best[:, 0] - best[:, 1] - 2e-6
    scores[::2, 1] += np.float32(4e-6)
    want = ref.select(x, scores.astype(np.float64), None, -1, 4)
    parent, token, score, _ = _run(g, dtype, logits, scores, None, -1, 4)
    assert [[(r[0], r[1]) for r in row] for row in want] == [[(int(a), int(b)) for a, b in zip(p, t)] for p, t in zip(parent, token)]
    w = np.array([[r[2] for r in row] for row in want])
    # one rounding to fp32, and the normaliser's stated bound
    assert np.all(np.abs(score - w) <= 2.0 ** -24 * np.abs(w) + 2.3e-6)


@pytest.mark.parametrize("log_vocab,fraction", [(22, 0.49), (22, -0.49), (20, 0.49)])
def test_select_many_small_exponentials_in_close_candidates(g, log_vocab, fraction):
    """A peak over 2^20 or 2^22 equal logits whose exponentials are 1.49 or 1.51 times 2^(log_vocab - 61), against a beam that has
    only its peak: sums as multiples of that step would be off by half a step for each of them."""
    vocab = 1 << log_vocab
    logits = np.full((1, 2, vocab), -np.inf, dtype=np.float32)
    term = (1.49 if fraction > 0 else 1.51) * 2.0 ** (log_vocab - 61)
    logits[0, 0], logits[0, :, 1000] = np.log(term), 0.0
    off = vocab * 0.49 * 2.0 ** (log_vocab - 61)
    best = -np.log1p((vocab - 1) * np.exp(np.float64(logits[0, 0, 0])))
    _check(g, 0, logits, np.array([[0.0, best + (off if fraction > 0 else -off) / 2]]), None, -1, 2)
