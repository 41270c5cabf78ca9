"""The paged key / value cache of batched decoding: appending with rotation, attention over a shared prefix and own rows, and
reordering of states, against plain 64-bit forms (tests/paged_ref.py)."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    from tests import gpu_util
    return gpu_util


def _torch_type(dtype):
    import torch
    return torch.bfloat16 if dtype else torch.float32


def _descr(g, kp, vp, page, dtype, layers=1):
    shape = kp.shape
    return g.nnb.PagedKv(kp.data_ptr(), vp.data_ptr(), kp.numel() // layers, layers, shape[-4], page, shape[-3], shape[-1], dtype)


def _f64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ append
def _append_case(g, dtype, src, heads, hk, dk, page, tokens, seqs, per, rope, with_q, ld_extra=0, offset=0, seed=0, rope_pos=False, bad=True):
    import torch
    r = np.random.default_rng(seed)
    pages = seqs * per + 2
    ts, td = _torch_type(src), _torch_type(dtype)
    width = (heads + 2 * hk) * dk + ld_extra
    flat = torch.from_numpy(r.standard_normal(tokens * width + offset).astype(np.float32)).cuda().to(ts)
    qkv = flat[offset:].view(tokens, width)
    kp, vp = (torch.from_numpy(r.standard_normal((pages, hk, page, dk)).astype(np.float32)).cuda().to(td) for _ in range(2))
    table = r.permutation(pages)[:seqs * per].reshape(seqs, per).astype(np.int32)
    places = r.permutation(seqs * per * page)[:tokens]                       # distinct (sequence, row) pairs
    seq_of, row_of = (places // (per * page)).astype(np.int32), (places % (per * page)).astype(np.int32)
    pos = r.integers(0, 50, tokens).astype(np.int32) if rope_pos else None
    rope_len = 50 if rope_pos else per * page
    if bad and tokens >= 12:
        # tokens that have no place: a padded one, a row behind the table, a sequence that is not there, pages that are not there
        row_of[0], row_of[1], seq_of[2], seq_of[3] = -1, per * page, -1, seqs
        seq_of[4], row_of[4], seq_of[5], row_of[5] = 0, 0, 0, page if per > 1 else 1
        table[0, 0] = -1
        if per > 1:
            table[0, 1] = pages
    rope_t = None
    if rope:
        ang = np.arange(rope_len)[:, None] / 10000.0 ** (2.0 * np.arange(dk // 2) / dk)
        rope_t = np.stack([np.cos(ang), np.sin(ang)]).astype(np.float32)
        rope_t = np.ascontiguousarray(rope_t)
        if not rope_pos and bad:
            rope_len = max(1, per * page - 2)                                # the last rows have no position
            rope_t = np.ascontiguousarray(rope_t[:, :rope_len])
    x = _f64(qkv)
    q, k, v = x[:, :heads * dk].reshape(tokens, heads, dk), x[:, heads * dk:(heads + hk) * dk].reshape(tokens, hk, dk), \
        x[:, (heads + hk) * dk:(heads + 2 * hk) * dk].reshape(tokens, hk, dk)
    want_k, want_v = _f64(kp), _f64(vp)
    want_q = ref.append(want_k, want_v, q if with_q else None, k, v, seq_of, row_of, table, rope_t, pos, page)
    q_out = torch.full((tokens, heads * dk + ld_extra), 7.0, device="cuda", dtype=td)
    es = qkv.element_size()
    base = qkv.data_ptr()
    keep = [g.dev(a) if a is not None else None for a in (seq_of, row_of, table, rope_t, pos)]
    kv = _descr(g, kp, vp, page, dtype)
    g.call("nnb200_paged_append", C.byref(kv), 0, base if with_q else None, width, q_out.data_ptr() if with_q else None, heads * dk + ld_extra, base + heads * dk * es,
           base + (heads + hk) * dk * es, width, src, tokens, heads, g.ptr(keep[0]), g.ptr(keep[1]), g.ptr(keep[2]), seqs, per, g.ptr(keep[3]), rope_len if rope else 0,
           g.ptr(keep[4]), g.stream())
    torch.cuda.synchronize()
    # two products and a sum of fp32, each half a step off (and |x c| + |y s| <= sqrt(2) |(x, y)|), then one rounding to the type
    def near(got, want):
        size = np.abs(want).max() if want.size else 0.0
        assert np.all(np.abs(got - want) <= ref.HALF_STEP[dtype] * np.abs(want) + (4 * ref.U * 1.5 * max(size, np.abs(x).max()) if rope else 0.0))
    near(_f64(kp), want_k)
    assert np.array_equal(_f64(vp), np.asarray(torch.from_numpy(want_v).to(td).double()))
    if with_q:
        got = _f64(q_out)
        assert np.all(got[:, heads * dk:] == 7.0)
        out = np.isnan(want_q).any(axis=(1, 2))
        assert np.all(got[out] == 7.0)
        near(got[~out, :heads * dk], want_q[~out].reshape(-1, heads * dk))
    else:
        assert np.all(_f64(q_out) == 7.0)


@pytest.mark.parametrize("dtype,src", [(0, 0), (1, 1), (1, 0), (0, 1)])
@pytest.mark.parametrize("heads,hk,dk,page", [(6, 6, 64, 16), (8, 2, 128, 64), (3, 1, 8, 8), (5, 5, 40, 32), (4, 4, 72, 8), (2, 2, 256, 256)])
@pytest.mark.parametrize("rope,with_q", [(True, True), (False, True), (True, False)])
def test_append(g, dtype, src, heads, hk, dk, page, rope, with_q):
    _append_case(g, dtype, src, heads, hk, dk, page, 37, 3, 2 if page == 256 else 5, rope, with_q)


@pytest.mark.parametrize("tokens", [1, 2, 1000])
def test_append_lengths(g, tokens):
    _append_case(g, 1, 1, 4, 2, 64, 16, tokens, 9, 12, True, True, bad=tokens > 2)


@pytest.mark.parametrize("dtype,src", [(0, 0), (1, 1), (1, 0)])
def test_append_odd_strides_and_positions_of_their_own(g, dtype, src):
    _append_case(g, dtype, src, 3, 3, 64, 16, 29, 2, 4, True, True, ld_extra=3, offset=1, rope_pos=True)
    _append_case(g, dtype, src, 3, 3, 64, 16, 29, 2, 4, True, True, ld_extra=8, rope_pos=True)


def test_append_in_place_and_without_seq_of(g):
    """Queries rotated where they are; token i to sequence i; in every layer's own pages."""
    import torch
    heads, dk, page, layers, tokens, per = 4, 64, 16, 3, 7, 2
    r = np.random.default_rng(3)
    qkv = torch.from_numpy(r.standard_normal((tokens, 3 * heads * dk)).astype(np.float32)).cuda()
    x = _f64(qkv).reshape(tokens, 3, heads, dk)
    kp, vp = (torch.zeros((layers, tokens * per, heads, page, dk), device="cuda") for _ in range(2))
    table = np.arange(tokens * per, dtype=np.int32).reshape(tokens, per)
    row = r.integers(0, per * page, tokens).astype(np.int32)
    rope = torch.empty(2 * 64 * dk // 2)
    g.call("nnb200_rope_table", 64, dk, C.c_void_p(rope.data_ptr()))
    want_k, want_v = np.zeros(kp.shape[1:]), np.zeros(kp.shape[1:])
    want_q = ref.append(want_k, want_v, x[:, 0], x[:, 1], x[:, 2], None, row, table, rope.double().numpy().reshape(2, 64, -1), None, page)
    kv = _descr(g, kp, vp, page, 0, layers)
    d = heads * dk
    t, ro, rp = g.dev(table), g.dev(row), rope.cuda()
    g.call("nnb200_paged_append", C.byref(kv), 2, g.ptr(qkv), 3 * d, g.ptr(qkv), 3 * d, C.c_void_p(qkv.data_ptr() + 4 * d), C.c_void_p(qkv.data_ptr() + 8 * d), 3 * d, 0, tokens,
           heads, None, g.ptr(ro), g.ptr(t), tokens, per, g.ptr(rp), 64, None, g.stream())
    torch.cuda.synchronize()
    assert not kp[:2].any() and not vp[:2].any()
    tol = 8 * ref.U * np.abs(x).max()
    assert np.abs(_f64(kp[2]) - want_k).max() <= tol and np.array_equal(_f64(vp[2]), want_v)
    got = _f64(qkv).reshape(tokens, 3, heads, dk)
    assert np.abs(got[:, 0] - want_q).max() <= tol and np.array_equal(got[:, 1:], x[:, 1:])


# ------------------------------------------------------------------------------------------------ attention
def _attention_inputs(dtype, heads, hk, dk, page, groups, size, prefix, own, seed=0, spread=1.0):
    """prefix, own: lengths per group and per sequence.  Rows that no query sees hold NaN, in pages that are used and others."""
    r = np.random.default_rng(seed)
    n = groups * size
    up = lambda m: -(-m // page)  # noqa: E731
    wide_p, wide_o = max([up(p) for p in prefix] + [0]), max([up(max(o, 0)) for o in own] + [0])
    pages = groups * wide_p + n * wide_o + 3
    order = r.permutation(pages).astype(np.int32)
    ptab, otab = order[:groups * wide_p].reshape(groups, wide_p), order[groups * wide_p:groups * wide_p + n * wide_o].reshape(n, wide_o)
    kp, vp = (np.full((pages, hk, page, dk), np.nan, np.float32) for _ in range(2))

    def fill(tab, count):
        for t in range(max(count, 0)):
            kp[tab[t // page], :, t % page] = r.standard_normal((hk, dk))
            vp[tab[t // page], :, t % page] = r.standard_normal((hk, dk))
    for i in range(groups):
        fill(ptab[i], prefix[i])
    for i in range(n):
        fill(otab[i], own[i])
    q = (spread * r.standard_normal((n, heads, dk))).astype(np.float32)
    return q, kp, vp, ptab, otab, np.array(prefix, np.int32), np.array(own, np.int32)


def _attention(g, dtype, q, kp, vp, ptab, plen, otab, olen, size, alibi, ld_extra=0, lse=True, scratch=None, fill=5.0):
    """Runs the entry point on tensors and returns (out, lse, the whole output buffer)."""
    import torch
    n, heads, dk = q.shape
    groups = n // size
    t = _torch_type(dtype)
    ld = heads * dk + ld_extra
    qd = torch.zeros((n, ld), device="cuda", dtype=t)
    qd[:, :heads * dk] = torch.from_numpy(q.reshape(n, -1)).cuda()
    out = torch.full((n + 2, ld), fill, device="cuda", dtype=t)
    ls = torch.full((n, heads), fill, device="cuda")
    kv = _descr(g, kp, vp, kp.shape[2], dtype)
    keep = [g.dev(a) for a in (ptab, plen, otab, olen)]
    need = g.call("nnb200_paged_attention_scratch_bytes", C.byref(kv), groups, size, heads, ptab.shape[1], otab.shape[1])
    if scratch is None:
        scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")           # NaN to whoever reads before writing
    g.call("nnb200_paged_attention", C.byref(kv), 0, g.ptr(qd), ld, C.c_void_p(out.data_ptr()), ld, g.ptr(ls) if lse else None, g.ptr(keep[0]) if ptab.size else None,
           ptab.shape[1], g.ptr(keep[1]), g.ptr(keep[2]) if otab.size else None, otab.shape[1], g.ptr(keep[3]), groups, size, heads, alibi, g.ptr(scratch), need, g.stream())
    torch.cuda.synchronize()
    assert bool((scratch[need:] == 255).all())
    assert bool((out[n:] == fill).all()) and bool((out[:, heads * dk:] == fill).all())
    return _f64(out[:n, :heads * dk]).reshape(n, heads, dk), _f64(ls), out


def _check_attention(g, dtype, heads, hk, dk, page, groups, size, prefix, own, alibi=0, seed=0, spread=1.0, ld_extra=0, change=None):
    import torch
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(dtype, heads, hk, dk, page, groups, size, prefix, own, seed, spread)
    t = _torch_type(dtype)
    if change:
        q, kp, vp, ptab, otab, plen, olen = change(q, kp, vp, ptab, otab, plen, olen)
    kt, vt = torch.from_numpy(kp).cuda().to(t), torch.from_numpy(vp).cuda().to(t)
    qr = torch.from_numpy(q).to(t)
    want, want_lse, tol, tol_lse = ref.attention(_f64(qr), _f64(kt), _f64(vt), ptab, plen, otab, olen, size, alibi, dtype)
    got, got_lse, _ = _attention(g, dtype, q, kt, vt, ptab, plen, otab, olen, size, alibi, ld_extra)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / np.maximum(tol, 1e-30)).max())
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(got_lse), empty)
    assert np.all(np.abs(got_lse[~empty] - want_lse[~empty]) <= tol_lse[~empty])


HEADS = [(6, 6, 64, 16), (8, 2, 128, 64), (3, 1, 8, 8), (5, 5, 40, 32), (4, 2, 72, 8), (2, 2, 256, 256), (2, 1, 136, 16), (12, 1, 32, 16), (40, 2, 96, 32)]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads,hk,dk,page", HEADS)
@pytest.mark.parametrize("alibi", [0, 1])
def test_attention_heads(g, dtype, heads, hk, dk, page, alibi):
    """Head layouts and page sizes: lengths that end inside pages and tiles, padded and empty sequences, an empty prefix."""
    _check_attention(g, dtype, heads, hk, dk, page, 3, 4, [83, 0, 1], [1, 17, -1, 64, 0, 1, 33, -1, 5, 0, 70, 2], alibi)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("size", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 97, 130, 161, 257])
def test_attention_group_sizes(g, dtype, size):
    """One sequence to more than two tiles of them behind one prefix."""
    own = [(7 * i) % 23 - 1 for i in range(size)]
    _check_attention(g, dtype, 2, 2, 64, 16, 1, size, [307], own, seed=size)
    _check_attention(g, dtype, 4, 1, 128, 32, 1, size, [130], own, seed=size, alibi=1)


@pytest.mark.parametrize("heads,hk,dk,page,size", [(4, 4, 64, 8, 90), (2, 2, 40, 128, 70), (8, 2, 128, 256, 20), (6, 2, 96, 8, 40), (4, 1, 72, 64, 5), (3, 1, 256, 16, 30),
                                                   (2, 2, 64, 256, 40), (32, 1, 128, 16, 9)])
@pytest.mark.parametrize("alibi", [0, 1])
def test_attention_many_rows(g, heads, hk, dk, page, size, alibi):
    """Tiles of every kind with page sizes below, at and above their boxes, heads that pad them, odd strides and missing pages."""
    prefix, own = [333, 128], [(11 * i) % 37 - 1 for i in range(2 * size)]
    _check_attention(g, 1, heads, hk, dk, page, 2, size, prefix, own, alibi, seed=size)
    _check_attention(g, 1, heads, hk, dk, page, 2, size, prefix, own, alibi, seed=size, ld_extra=3)

    def change(q, kp, vp, ptab, otab, plen, olen):
        ptab[0, min(1, ptab.shape[1] - 1)], ptab[1, 0], otab[3, 0] = -1, kp.shape[0], 2 ** 31 - 1
        return q, kp, vp, ptab, otab, plen, olen
    _check_attention(g, 1, heads, hk, dk, page, 2, size, prefix, own, alibi, seed=size, change=change)


@pytest.mark.parametrize("heads,hk,dk,size", [(24, 12, 80, 20), (12, 12, 128, 17), (12, 12, 64, 66)])
def test_attention_of_some_rows_behind_runs_of_several_steps(g, heads, hk, dk, size):
    """Tiles that are not full of queries, runs of several steps that end inside one."""
    own = [(5 * i) % 9 for i in range(size)]
    _check_attention(g, 1, heads, hk, dk, 64, 1, size, [6300], own, seed=size)
    _check_attention(g, 1, heads, hk, dk, 16, 1, size, [7003], own, alibi=1, seed=size)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads,hk,dk,groups,size", [(16, 16, 40, 3, 50), (40, 2, 32, 2, 33)])
def test_attention_of_more_query_rows_than_are_joined_at_a_time(g, dtype, heads, hk, dk, groups, size):
    own = [(13 * i) % 150 - 1 for i in range(groups * size)]
    _check_attention(g, dtype, heads, hk, dk, 16, groups, size, [300, 0, 77][:groups], own, seed=heads)


def test_attention_of_many_rows_large_scores_and_status_word(g):
    _check_attention(g, 1, 4, 4, 64, 16, 1, 100, [1500], [(7 * i) % 50 for i in range(100)], seed=9, spread=60.0)
    _check_attention(g, 1, 8, 2, 128, 32, 1, 30, [1500], [(7 * i) % 50 for i in range(30)], seed=9, spread=60.0)
    assert g.gemm_status() == 0


@pytest.mark.parametrize("heads,hk,dk,size", [(2, 2, 64, 90), (4, 1, 128, 20), (2, 2, 64, 30), (2, 2, 64, 5)])
@pytest.mark.parametrize("prefix,own", [([700], 21), ([200], 0)])
def test_attention_scores_of_hundreds_of_thousands(g, heads, hk, dk, size, prefix, own):
    """Scores of 2e4 to 7e5 of either sign, that differ by little: column 0 gives all of a query's scores one large number, the
    others whole numbers.  Products and partial sums are whole numbers below 2^24, exact in fp32 in whatever order, so the
    weights depend only on differences of tens, whose scaling is off by 2^-24 twice: the large number is the same in every one."""
    import torch
    n = size
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(1, heads, hk, dk, 16, 1, size, prefix, [(7 * i) % (own + 1) for i in range(n)], dk + size)
    r = np.random.default_rng(3)
    kp = np.where(np.isnan(kp), kp, r.integers(-2, 3, kp.shape)).astype(np.float32)
    q = r.integers(-2, 3, q.shape).astype(np.float32)
    kp[..., 0] = np.where(np.isnan(kp[..., 0]), np.nan, 128.0)
    q[..., 0] = 2.0 ** r.integers(11, 16, q.shape[:2]) * r.choice([-1.0, 1.0], q.shape[:2])
    q[0, 0, 0], q[1, 0, 0] = 2.0 ** 15, -2.0 ** 15
    kt, vt = torch.from_numpy(kp).cuda().bfloat16(), torch.from_numpy(vp).cuda().bfloat16()
    want, want_lse, _, _ = ref.attention(q.astype(np.float64), _f64(kt), _f64(vt), ptab, plen, otab, olen, size, 0, 1)
    size_v, _, _, _ = ref.attention(q.astype(np.float64), _f64(kt), np.abs(_f64(vt)), ptab, plen, otab, olen, size, 0, 1)
    got, got_lse, _ = _attention(g, 1, q, kt, vt, ptab, plen, otab, olen, size, 0)
    # differences of at most 2 * 4 * dk / sqrt(dk) * log2(e) in powers of two, rounded with the factor and with the sum; an exponential
    # 4 steps, sums of `total` terms; the weight's and the result's rounding to bf16
    total = prefix[0] + own
    weight = 2 * (2 * 8 * np.sqrt(dk) * 1.45 * ref.U + 4 * ref.U) + 2 * (total + 40) * ref.U + ref.HALF_STEP[1]
    assert np.all(np.abs(got - want) <= weight * size_v + ref.HALF_STEP[1] * np.abs(want) + 1e-37), float(np.abs(got - want).max())
    assert np.all(np.abs(got_lse - want_lse) <= 6 * ref.U * np.abs(want_lse) + (total + 40) * ref.U + 1e-4)
    assert g.gemm_status() == 0


@pytest.mark.parametrize("heads,hk,dk,size", [(2, 2, 64, 80), (4, 1, 128, 40), (2, 2, 64, 30), (1, 1, 256, 20)])
def test_attention_of_many_rows_meets_infinities(g, heads, hk, dk, size):
    """A key of -inf has no weight, a value of +inf is one column's, a NaN key everybody's that sees it."""
    import torch
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(1, heads, hk, dk, 16, 2, size, [200, 77], [3] * (2 * size), 4)
    q = np.abs(q) + 0.01
    run = lambda k, v: _attention(g, 1, q, torch.from_numpy(k).cuda().bfloat16(), torch.from_numpy(v).cuda().bfloat16(), ptab, plen, otab, olen, size, 0)  # noqa: E731
    clean, clean_lse, _ = run(kp, vp)
    k2, v2 = kp.copy(), vp.copy()
    k2[ptab[0, 2], :, 5] = -np.inf
    v2[ptab[0, 0], :, 1, 7] = np.inf
    got, lse, _ = run(k2, v2)
    assert np.array_equal(got[size:], clean[size:]) and np.array_equal(lse[size:], clean_lse[size:])
    assert np.all(got[:size, :, 7] == np.inf) and np.isfinite(np.delete(got[:size], 7, 2)).all() and np.all(lse[:size] < clean_lse[:size])
    k2[ptab[0, 1], :, 0, 0] = np.nan
    got, lse, _ = run(k2, vp)
    assert np.isnan(got[:size]).all() and np.isnan(lse[:size]).all() and np.array_equal(got[size:], clean[size:])
    got, lse, _ = run(np.where(np.isnan(kp), kp, -np.inf).astype(np.float32), vp)
    assert np.all(got == 0) and np.all(np.isneginf(lse))


def test_attention_on_two_streams_at_once(g):
    """Two calls that may overlap, each with a scratch of its own; tensors made on one stream and used on another behind it."""
    import torch
    cases = []
    for seed, (heads, hk, dk, size) in enumerate([(4, 4, 64, 90), (8, 2, 128, 3)]):
        q, kp, vp, ptab, otab, plen, olen = _attention_inputs(1, heads, hk, dk, 16, 2, size, [700, 333], [(13 * i) % 60 - 1 for i in range(2 * size)], seed)
        n = 2 * size
        t = dict(q=torch.from_numpy(q.reshape(n, -1)).cuda().bfloat16(), k=torch.from_numpy(kp).cuda().bfloat16(), v=torch.from_numpy(vp).cuda().bfloat16(), size=size, heads=heads)
        t.update(pt=g.dev(ptab), pl=g.dev(plen), ot=g.dev(otab), ol=g.dev(olen), out=torch.zeros((n, heads * dk), device="cuda", dtype=torch.bfloat16))
        t["kv"] = _descr(g, t["k"], t["v"], 16, 1)
        t["need"] = g.call("nnb200_paged_attention_scratch_bytes", C.byref(t["kv"]), 2, size, heads, ptab.shape[1], otab.shape[1])
        t["scratch"] = torch.empty(t["need"], dtype=torch.uint8, device="cuda")
        cases.append(t)

    def run(t):
        ld = t["q"].shape[1]
        g.call("nnb200_paged_attention", C.byref(t["kv"]), 0, g.ptr(t["q"]), ld, g.ptr(t["out"]), ld, None, g.ptr(t["pt"]), t["pt"].shape[1], g.ptr(t["pl"]), g.ptr(t["ot"]),
               t["ot"].shape[1], g.ptr(t["ol"]), 2, t["size"], t["heads"], 0, g.ptr(t["scratch"]), t["need"], g.stream())
        return t["out"]
    want = [run(t).clone() for t in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for s, t in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                run(t)
    torch.cuda.synchronize()
    assert all(torch.equal(t["out"], w) for t, w in zip(cases, want))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("prefix", [1, 7, 8, 63, 64, 65, 127, 128, 129, 1000, 4097])
def test_attention_prefix_lengths(g, dtype, prefix):
    _check_attention(g, dtype, 4, 4, 64, 16, 2, 3, [prefix, max(1, prefix - 1)], [3, 40, -1, 0, 1, 129], seed=prefix)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("own", [1, 16, 65, 1024, 5003])
def test_attention_without_prefix(g, dtype, own):
    _check_attention(g, dtype, 4, 2, 64, 32, 1, 3, [0], [own, 1, own - 1], alibi=1, seed=own)


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_without_own_rows(g, dtype):
    """No page table of their own at all: queries over the prefix alone, but for the padded one."""
    _check_attention(g, dtype, 4, 2, 64, 32, 2, 3, [100, 33], [0, 0, -1, 0, 0, 0])


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_of_nothing(g, dtype):
    _check_attention(g, dtype, 2, 2, 64, 16, 2, 2, [0, 0], [0, -1, -1, 0])
    _check_attention(g, dtype, 2, 2, 64, 16, 2, 2, [40, 0], [-1, -1, -1, 0])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads,hk,dk,page", [(6, 6, 64, 16), (8, 2, 128, 8), (3, 1, 40, 32), (40, 2, 32, 16), (2, 2, 256, 8)])
@pytest.mark.parametrize("alibi", [0, 1])
def test_attention_short_contexts(g, dtype, heads, hk, dk, page, alibi):
    """Prefix and own rows of a few steps together: lengths of nothing and one, padded sequences, both runs ending inside a step."""
    _check_attention(g, dtype, heads, hk, dk, page, 3, 4, [41, 0, 1], [1, 17, -1, 24, 0, 1, 16, -1, 5, 0, 23, 2], alibi)
    _check_attention(g, dtype, heads, hk, dk, page, 1, 2, [64], [64, 33], alibi, seed=1)

    def change(q, kp, vp, ptab, otab, plen, olen):
        ptab[0, 0], otab[1, 0] = -1, kp.shape[0]
        return q, kp, vp, ptab, otab, plen, olen
    _check_attention(g, dtype, heads, hk, dk, page, 1, 2, [40], [9, 30], alibi, seed=2, change=change)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads,hk,dk,page", [(6, 6, 64, 16), (8, 2, 128, 8), (3, 1, 40, 8), (40, 2, 32, 16), (2, 2, 256, 8)])
@pytest.mark.parametrize("prefix,own", [([33, 0, 1], [15, 0, -1, 1, 16, 2]), ([170, 9, 128], [1, 33, -1, 0, 64, 49])])
def test_attention_short_prefixes_and_own_rows(g, dtype, heads, hk, dk, page, prefix, own):
    _check_attention(g, dtype, heads, hk, dk, page, 3, 2, prefix, own, seed=3)
    _check_attention(g, dtype, heads, hk, dk, page, 3, 2, prefix, own, alibi=1, seed=4, ld_extra=3)


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_large_scores(g, dtype):
    """Scores of hundreds: weights of almost nothing and almost everything, maxima that move from tile to tile."""
    _check_attention(g, dtype, 4, 4, 64, 16, 1, 5, [700], [50, 1, 0, 300, 7], seed=9, spread=60.0)


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_odd_strides(g, dtype):
    _check_attention(g, dtype, 3, 3, 40, 16, 1, 5, [70], [5, 1, 0, 30, 7], ld_extra=3)
    _check_attention(g, dtype, 2, 2, 64, 16, 1, 5, [70], [5, 1, 0, 30, 7], ld_extra=1)


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_pages_that_are_not_there_and_lengths_beyond_the_tables(g, dtype):
    def change(q, kp, vp, ptab, otab, plen, olen):
        ptab[0, 2], ptab[1, 0] = -1, kp.shape[0]
        otab[0, 0], otab[4, 1], otab[5, :] = 2 ** 31 - 1, -2 ** 31, -5
        plen[1], olen[2] = 2 ** 31 - 1, 2 ** 31 - 1
        olen[3] = -2 ** 31
        for tab, ln in ((ptab, plen), (otab, olen)):        # what is visible now must be numbers
            for i in range(tab.shape[0]):
                for p in tab[i] if ln[i] > 100000 else []:
                    if 0 <= p < kp.shape[0]:
                        kp[p], vp[p] = np.nan_to_num(kp[p]), np.nan_to_num(vp[p])
        return q, kp, vp, ptab, otab, plen, olen
    _check_attention(g, dtype, 4, 2, 64, 16, 2, 3, [100, 100], [40, 3, 33, 20, 50, 17], change=change)


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_infinities_reach_only_who_sees_them(g, dtype):
    """An infinite or NaN row of one sequence leaves the others as they are; a key that gives -inf has no weight; a query whose
    every score is -inf gives 0 and -inf."""
    import torch
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(dtype, 2, 2, 64, 16, 1, 6, [90], [20] * 6, 4)
    t = _torch_type(dtype)
    q = np.abs(q)
    base = [torch.from_numpy(a).cuda().to(t) for a in (kp, vp)]
    clean, clean_lse, _ = _attention(g, dtype, q, *base, ptab, plen, otab, olen, 6, 0)
    k2, v2 = kp.copy(), vp.copy()
    k2[otab[1, 0], :, 3] = -np.inf                                  # a score of -inf
    v2[otab[2, 0], :, 3, 5] = np.inf
    v2[otab[3, 1], :, 2] = np.nan
    k2[otab[4, 0], :, 0] = np.nan
    got, got_lse, _ = _attention(g, dtype, q, *[torch.from_numpy(a).cuda().to(t) for a in (k2, v2)], ptab, plen, otab, olen, 6, 0)
    assert np.array_equal(got[[0, 5]], clean[[0, 5]]) and np.array_equal(got_lse[[0, 5]], clean_lse[[0, 5]])
    assert np.isfinite(got[1]).all() and np.all(got_lse[1] < clean_lse[1])
    assert np.all(got[2][:, 5] == np.inf) and np.array_equal(np.delete(got[2], 5, 1), np.delete(clean[2], 5, 1))
    assert np.isnan(got[3]).all() and np.array_equal(got_lse[3], clean_lse[3])
    assert np.isnan(got[4]).all() and np.isnan(got_lse[4]).all()
    k3 = np.where(np.isnan(kp), kp, -np.inf).astype(np.float32)
    got, got_lse, _ = _attention(g, dtype, q, torch.from_numpy(k3).cuda().to(t), base[1], ptab, plen, otab, olen, 6, 0)
    assert np.all(got == 0) and np.all(np.isneginf(got_lse))


@pytest.mark.parametrize("dtype", [0, 1])
def test_attention_without_lse_and_again_gives_the_same_bits(g, dtype):
    import torch
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(dtype, 8, 4, 64, 16, 2, 9, [900, 513], [(37 * i) % 200 for i in range(18)], 6)
    t = _torch_type(dtype)
    kt, vt = torch.from_numpy(kp).cuda().to(t), torch.from_numpy(vp).cuda().to(t)
    a, al, _ = _attention(g, dtype, q, kt, vt, ptab, plen, otab, olen, 9, 1)
    b, bl, _ = _attention(g, dtype, q, kt, vt, ptab, plen, otab, olen, 9, 1)
    c, cl, _ = _attention(g, dtype, q, kt, vt, ptab, plen, otab, olen, 9, 1, lse=False)
    assert np.array_equal(a, b) and np.array_equal(al, bl) and np.array_equal(a, c) and np.all(cl == 5.0)


def test_attention_offsets_beyond_32_bits(g):
    """A pool of more than 2^31 values, read at its far end."""
    import torch
    hk, dk, page = 8, 128, 64
    pages = (1 << 31) // (hk * dk * page) + 40
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(1, 8, hk, dk, page, 1, 4, [300], [70, 1, -1, 130], 8)
    kt, vt = (torch.zeros((pages, hk, page, dk), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    far = pages - kp.shape[0]
    kt[far:], vt[far:] = torch.from_numpy(kp).cuda().to(torch.bfloat16), torch.from_numpy(vp).cuda().to(torch.bfloat16)
    near_k, near_v = kt[far:].clone(), vt[far:].clone()
    want, want_lse, tol, tol_lse = ref.attention(_f64(torch.from_numpy(q).to(torch.bfloat16)), _f64(near_k), _f64(near_v), ptab, plen, otab, olen, 4, 0, 1)
    got, got_lse, _ = _attention(g, 1, q, kt, vt, ptab + np.int32(far), plen, otab + np.int32(far), olen, 4, 0)
    assert np.all(np.abs(got - want) <= tol)
    live = want_lse > -np.inf
    assert np.all(np.abs(got_lse[live] - want_lse[live]) <= tol_lse[live])


def test_attention_captured_and_replayed_with_new_lengths(g):
    """Lengths, page tables and queries are read when the graph runs, not when it is captured."""
    import torch
    dtype, size = 1, 5
    q, kp, vp, ptab, otab, plen, olen = _attention_inputs(dtype, 4, 4, 64, 16, 2, size, [300, 257], [90] * 10, 12)
    kt, vt = torch.from_numpy(kp).cuda().bfloat16(), torch.from_numpy(vp).cuda().bfloat16()
    qd = torch.from_numpy(q.reshape(10, -1)).cuda().bfloat16()
    out = torch.zeros_like(qd)
    kv = _descr(g, kt, vt, 16, dtype)
    pt, pl, ot, ol = (torch.from_numpy(a).cuda() for a in (ptab, plen, otab, olen))
    need = g.call("nnb200_paged_attention_scratch_bytes", C.byref(kv), 2, size, 4, ptab.shape[1], otab.shape[1])
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")

    def run():
        g.call("nnb200_paged_attention", C.byref(kv), 0, g.ptr(qd), 256, g.ptr(out), 256, None, g.ptr(pt), ptab.shape[1], g.ptr(pl), g.ptr(ot), otab.shape[1], g.ptr(ol), 2,
               size, 4, 0, g.ptr(scratch), need, g.stream())
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    r = np.random.default_rng(0)
    for _ in range(3):
        pl.copy_(torch.from_numpy(r.integers(0, 257, 2).astype(np.int32)))
        ol.copy_(torch.from_numpy(r.integers(-1, 91, 10).astype(np.int32)))
        qd.copy_(torch.from_numpy(r.standard_normal((10, 256)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        run()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        want, _, tol, _ = ref.attention(_f64(qd).reshape(10, 4, 64), _f64(kt), _f64(vt), ptab, _f64(pl).astype(int), otab, _f64(ol).astype(int), size, 0, dtype)
        assert np.all(np.abs(_f64(out).reshape(10, 4, 64) - want) <= tol)


# ------------------------------------------------------------------------------------------------ reorder
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("groups,beams,length,page,per", [(1, 1, 5, 8, 2), (2, 4, 37, 16, 4), (1, 8, 32, 16, 3), (3, 5, 0, 8, 2), (2, 3, 64, 32, 2), (1, 64, 9, 8, 2), (2, 2, 4, 8, 0)])
@pytest.mark.parametrize("hk,dk,layers", [(2, 64, 3), (1, 40, 1), (5, 8, 2)])
def test_reorder(g, dtype, groups, beams, length, page, per, hk, dk, layers):
    import torch
    r = np.random.default_rng(groups * 100 + beams)
    n = groups * beams
    pages = n * (per + 1)
    order = r.permutation(pages).astype(np.int32)
    table, spare = order[:n * per].reshape(n, per), order[n * per:].copy()
    parent = r.integers(0, beams, n).astype(np.int32)
    if n > 3:
        parent[1], parent[2] = -1, beams                       # out of range: stays with its own state
        if per:
            spare[3] = pages if groups == 2 else -1            # a page that is not there is not written
    lens = np.full(n, length, np.int32)
    if groups == 2:
        lens[beams:] = max(0, length - 3)                      # groups of unlike lengths
    t = _torch_type(dtype)
    kt, vt = (torch.from_numpy(r.standard_normal((layers, pages, hk, page, dk)).astype(np.float32)).cuda().to(t) for _ in range(2))
    want_k, want_v = _f64(kt), _f64(vt)
    want = ref.reorder(want_k, want_v, parent, lens, table, spare, beams)
    dev = [g.dev(a) for a in (parent, lens, table, spare)]
    outs = [torch.full((m + 3,), -7, dtype=torch.int32, device="cuda") for m in (n, n * per, n)]
    kv = _descr(g, kt, vt, page, dtype, layers)
    kv.pages = pages
    g.call("nnb200_beam_reorder", C.byref(kv), groups, beams, *[g.ptr(d) if d.numel() else None for d in dev], *[g.ptr(o) for o in outs], per, g.stream())
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o[:w.size].cpu().numpy(), w.reshape(-1)) and bool((o[w.size:] == -7).all())
    assert np.array_equal(_f64(kt), want_k) and np.array_equal(_f64(vt), want_v)
