"""Several continuations of a prompt together (nnb200_gpt_batch_*, GptTrainer.generate_beam) against the same tokens one sequence
at a time (nnb200_gpt_forward_step, which test_gpu_decode.py holds against the reference)."""
import ctypes as C

import numpy as np
import pytest

from oracle import gpt_oracle as go
from tests.golden_io import rel_err

pytestmark = pytest.mark.gpu


def _trainer(nnb, vocab, d, heads, layers, ff, seq, act, norm, pos, precision, std=0.05):
    tr = nnb.GptTrainer(nnb.GptConfig(vocab, d, heads, layers, ff, seq, 1, act, norm, pos, precision))
    tr.load_params(go.init_params(go.GptConfig(vocab, d, heads, layers, ff, seq, 1, act, norm, pos), 5, std=std))
    return tr


# (heads, head size, seq, prompt, sequences, new rows): pages that end inside tiles, a prompt shorter than a page and one over
# many, a head size that pads its tile, one sequence and more than a tile of them
SHAPES = [(2, 32, 80, 5, 3, 19), (3, 64, 300, 257, 5, 21), (1, 128, 131, 90, 17, 4), (2, 24, 40, 20, 1, 18), (2, 64, 64, 33, 40, 3)]


@pytest.mark.parametrize("heads,dk,seq,n,seqs,new", SHAPES)
@pytest.mark.parametrize("act,norm,pos", [(0, 0, 0), (1, 1, 2), (1, 1, 3), (1, 0, 1)])
@pytest.mark.parametrize("precision", [0, 1])
def test_steps_of_several_sequences_equal_single_ones(heads, dk, seq, n, seqs, new, act, norm, pos, precision):
    """Tokens drawn at random, the states reordered before every second one: the logits of each sequence are those of a decoding
    that has run its tokens alone."""
    import torch
    from tests import gpu_util as g
    tr = _trainer(g.nnb, 72, heads * dk, heads, 2, 104, seq, act, norm, pos, precision)
    r = np.random.default_rng(seqs)
    prompt = [int(t) for t in r.integers(0, 72, n)]
    tr.prefill(prompt)
    dec, _ = tr._decode_state()
    size = g.call("nnb200_gpt_batch_workspace_bytes", C.byref(tr._c), seqs, new)
    ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")         # NaN to whoever reads before writing
    logits = torch.empty((seqs, 72), device="cuda")
    g.call("nnb200_gpt_batch_begin", C.byref(tr._c), g.ptr(dec), g.ptr(ws), seqs, new, n, g.stream())
    history, got = [list(prompt) for _ in range(seqs)], None
    for step in range(new):
        if step % 2:
            parent = r.integers(-1, seqs + 1, seqs).astype(np.int32)
            g.call("nnb200_gpt_batch_reorder", C.byref(tr._c), g.ptr(ws), seqs, new, g.ptr(g.dev(parent)), g.stream())
            history = [list(history[p if 0 <= p < seqs else i]) for i, p in enumerate(parent)]
        tokens = r.integers(0, 72, seqs).astype(np.int32)
        for i, t in enumerate(tokens):
            history[i].append(int(t))
        g.call("nnb200_gpt_batch_step", C.byref(tr._c), g.ptr(tr.params), g.ptr(tr.shadow), g.ptr(dec), g.ptr(ws), seqs, new, n, step, g.ptr(g.dev(tokens)), g.ptr(logits),
               g.stream())
    torch.cuda.synchronize()
    assert bool((ws[size:] == 255).all())
    got = logits.cpu().numpy()
    for i in sorted({0, seqs // 2, seqs - 1}):
        for t, tok in enumerate(history[i]):
            if t >= n - 1 or i == 0:                             # the prompt's rows are in the cache already
                want = tr.forward_step(tok, t, t)
        # fp32 sums of up to 300 terms in another order through two layers: n eps / 2 at most, their square root in practice
        assert rel_err(got[i], want.cpu().numpy()) < 1e-5


def _beam_by_steps(tr, prompt, beams, new, eos):
    """Beam search on the host, in 64 bits, from single steps: [(tokens, score)], best first."""
    def log_probs(tokens):
        if len(tokens) == len(prompt):
            x = tr.prefill(prompt)
        else:
            for t in range(len(prompt), len(tokens)):
                x = tr.forward_step(tokens[t], t, t)
        x = x.double().cpu().numpy()
        return x - x.max() - np.log(np.exp(x - x.max()).sum())
    live = [(list(prompt), 0.0, False)]
    for _ in range(new):
        cand = []
        for b, (tokens, score, ended) in enumerate(live):
            if ended:
                cand.append((-score, b, eos, tokens, True))
                continue
            lp = log_probs(tokens)
            cand += [(-(score + lp[t]), b, t, tokens, t == eos) for t in range(len(lp))]
        cand.sort(key=lambda c: c[:3])
        live = [(c[3] + [c[2]], -c[0], c[4]) for c in cand[:beams]]
        if all(e for _, _, e in live):
            break
    out = []
    for tokens, score, _ in live:
        tokens = tokens[len(prompt):]
        out.append((tokens[:tokens.index(eos)] if eos in tokens else tokens, score))
    return out


@pytest.mark.parametrize("pos,precision,beams,n,new", [(2, 0, 4, 9, 12), (3, 1, 5, 40, 20), (0, 0, 1, 3, 6), (1, 1, 8, 17, 17), (3, 0, 64, 12, 3)])
@pytest.mark.parametrize("eos", [-1, 7])
def test_beam_search_finds_what_single_steps_find(pos, precision, beams, n, new, eos):
    from tests.gpu_util import nnb
    tr = _trainer(nnb, 80, 128, 2, 2, 104, 64, 1, 1, pos, precision, std=0.3)
    prompt = [int(t) for t in np.random.default_rng(n).integers(0, 80, n)]
    got = tr.generate_beam(prompt, beams, new, eos_token_id=eos)
    want = _beam_by_steps(tr, prompt, beams, new, eos)
    # scores sum up to `new` log-probabilities of logits that are 1e-5 of their size apart
    assert [t for t, _ in got] == [t for t, _ in sorted(want, key=lambda w: -w[1])]
    assert np.allclose([s for _, s in got], [s for _, s in sorted(want, key=lambda w: -w[1])], rtol=1e-4, atol=1e-3)


def test_one_beam_is_greedy_and_length_penalty_orders():
    from tests.gpu_util import nnb
    tr = _trainer(nnb, 72, 64, 2, 2, 104, 96, 1, 1, 2, 0, std=0.3)
    prompt = [3, 5, 7, 11, 13]
    assert tr.generate_beam(prompt, 1, 30)[0][0] == tr.generate(prompt, 30, temperature=0.0)
    plain, long = tr.generate_beam(prompt, 6, 8, eos_token_id=9), tr.generate_beam(prompt, 6, 8, eos_token_id=9, length_penalty=5.0)
    assert sorted(plain) == sorted(long)
    assert [s / max(1, len(t)) ** 5.0 for t, s in long] == sorted((s / max(1, len(t)) ** 5.0 for t, s in long), reverse=True)


def test_beam_search_leaves_decoding_as_it_was():
    """The decode cache holds the prompt afterwards, and the next search is the same."""
    import torch
    from tests.gpu_util import nnb
    tr = _trainer(nnb, 72, 64, 2, 2, 104, 96, 1, 1, 3, 1)
    prompt = list(range(20))
    want = tr.prefill(prompt).clone()
    behind = tr.forward_step(5, 20, 20).clone()
    a = tr.generate_beam(prompt, 4, 10)
    assert torch.equal(tr.forward_step(5, 20, 20), behind) and a == tr.generate_beam(prompt, 4, 10)
    assert torch.equal(tr.prefill(prompt), want)


def test_beam_search_refuses():
    from tests.gpu_util import nnb
    tr = _trainer(nnb, 72, 64, 2, 1, 104, 32, 1, 1, 3, 1)
    for args in (([], 2, 4), ([1], 0, 4), ([1], 65, 4), ([1], 2, 0), ([1] * 30, 2, 3)):
        with pytest.raises(ValueError):
            tr.generate_beam(*args)
    for eos in (-2, 72):
        with pytest.raises(ValueError):
            tr.generate_beam([1, 2], 2, 4, eos_token_id=eos)
