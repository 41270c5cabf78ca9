"""Arguments that the batched-decoding entry points refuse.  The checks are the host's, so no GPU is needed: the pointers are
never followed."""
import ctypes as C

import pytest

import __graft_entry__ as entry

nnb = entry.load_package()
P = 1 << 20                                        # an aligned address that nothing reads


def kv(**change):
    a = dict(k=P, v=P, layer_stride=64 * 2 * 16 * 64, layers=2, pages=64, page_size=16, kv_heads=2, head_dim=64, dtype=1)
    a.update(change)
    return nnb.PagedKv(*(a[f] for f, _ in nnb.PagedKv._fields_[:-1]))


BAD_KV = [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(layers=0), dict(pages=0), dict(pages=-1), dict(page_size=4), dict(page_size=24),
          dict(page_size=512), dict(page_size=0), dict(kv_heads=0), dict(kv_heads=65536), dict(head_dim=4), dict(head_dim=60), dict(head_dim=264), dict(head_dim=0),
          dict(dtype=2), dict(dtype=-1), dict(layer_stride=64 * 2 * 16 * 64 - 8), dict(layer_stride=64 * 2 * 16 * 64 + 4)]


def refused(name, *args):
    assert getattr(nnb.lib, name)(*args) == -1
    with pytest.raises(nnb.NnbError):
        nnb.call(name, *args)


def append_args(kv_=None, **change):
    a = dict(layer=0, q=P, ldq=512, q_out=2 * P, ldqo=256, k=P, v=P, ldkv=512, src_dtype=1, tokens=3, heads=4, seq_of=P, row_of=P, table=P, seqs=3, stride=4, rope=P,
             rope_len=64, rope_pos=None, stream=None)
    a.update(change)
    return (C.byref(kv_ or kv()), *a.values())


@pytest.mark.parametrize("change", [dict(layer=-1), dict(layer=2), dict(src_dtype=2), dict(tokens=-1), dict(heads=-1), dict(seqs=-1), dict(stride=-1), dict(k=None),
                                    dict(v=None), dict(row_of=None), dict(table=None), dict(q=None), dict(q_out=None), dict(heads=0), dict(seq_of=None, tokens=4),
                                    dict(ldkv=127), dict(ldq=255), dict(ldqo=255), dict(q_out=P), dict(q_out=P, ldqo=512, src_dtype=0), dict(rope_len=0),
                                    dict(stride=1 << 28), dict(heads=1 << 20)])
def test_append_refuses(change):
    refused("nnb200_paged_append", *append_args(**change))


def attention_args(kv_=None, **change):
    a = dict(layer=0, q=P, ldq=256, out=P, ldo=256, lse=None, prefix_table=P, prefix_stride=4, prefix_len=P, table=P, stride=2, len=P, groups=2, size=3, heads=4, alibi=0,
             scratch=P, scratch_bytes=1 << 40, stream=None)
    a.update(change)
    return (C.byref(kv_ or kv()), *a.values())


@pytest.mark.parametrize("change", [dict(layer=-1), dict(layer=2), dict(q=None), dict(out=None), dict(len=None), dict(prefix_table=None), dict(prefix_len=None),
                                    dict(table=None), dict(ldq=255), dict(ldo=0), dict(heads=0), dict(heads=3), dict(heads=-2), dict(groups=-1), dict(size=-1),
                                    dict(prefix_stride=-1), dict(stride=-1), dict(scratch=None), dict(scratch=P + 8), dict(scratch_bytes=0),
                                    dict(groups=1 << 15, size=1 << 15), dict(stride=1 << 28), dict(prefix_stride=1 << 28)])
def test_attention_refuses(change):
    refused("nnb200_paged_attention", *attention_args(**change))


def select_args(**change):
    a = dict(logits=P, ld=100, dtype=0, groups=2, beams=4, vocab=100, scores=P, ended=P, eos=2, n=8, parent=P, token=P, scores_out=P, ended_out=P, scratch=P,
             scratch_bytes=1 << 40, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize("change", [dict(logits=None), dict(ld=99), dict(dtype=2), dict(groups=-1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(scores=None),
                                    dict(eos=-1), dict(eos=100), dict(n=0), dict(n=129), dict(beams=1, vocab=5, ld=5, n=6), dict(parent=None), dict(token=None),
                                    dict(scores_out=None), dict(scratch=None), dict(scratch=P + 4), dict(scratch_bytes=15), dict(vocab=1 << 30, ld=1 << 30),
                                    dict(groups=1 << 24)])
def test_select_refuses(change):
    refused("nnb200_beam_select", *select_args(**change))


@pytest.mark.parametrize("vocab", [2 ** 31 - 1, 2 ** 31 - 2 ** 16])
def test_select_refuses_vocabularies_whose_last_tile_ends_beyond_32_bits(vocab):
    """A block reads spans of up to 2^16 logits and counts tokens in 32 bits to the end of the last one."""
    assert nnb.lib.nnb200_beam_select_scratch_bytes(1, 1, vocab, 4) == 0
    refused("nnb200_beam_select", *select_args(groups=1, beams=1, vocab=vocab, ld=vocab, n=4))
    assert nnb.lib.nnb200_beam_select_scratch_bytes(1, 1, 2 ** 31 - 2 ** 16 - 1, 4) > 0
    assert nnb.lib.nnb200_beam_select_scratch_bytes(1, 63, (2 ** 31 - 1) // 63, 4) > 0


def reorder_args(kv_=None, **change):
    a = dict(groups=2, beams=3, parent=P, len=P, table=P, spare=P, len_out=2 * P, table_out=2 * P, spare_out=2 * P, stride=4, stream=None)
    a.update(change)
    return (C.byref(kv_ or kv()), *a.values())


@pytest.mark.parametrize("change", [dict(groups=-1), dict(beams=-1), dict(stride=-1), dict(parent=None), dict(len=None), dict(table=None), dict(spare=None),
                                    dict(len_out=None), dict(table_out=None), dict(spare_out=None), dict(len_out=P), dict(table_out=P), dict(spare_out=P),
                                    dict(groups=1 << 16, beams=1 << 16), dict(stride=1 << 28)])
def test_reorder_refuses(change):
    refused("nnb200_beam_reorder", *reorder_args(**change))


@pytest.mark.parametrize("change", BAD_KV)
def test_bad_cache_descriptions_are_refused(change):
    bad = kv(**change)
    refused("nnb200_paged_append", *append_args(bad))
    refused("nnb200_paged_attention", *attention_args(bad))
    refused("nnb200_beam_reorder", *reorder_args(bad))
    assert nnb.lib.nnb200_paged_attention_scratch_bytes(C.byref(bad), 2, 3, 4, 4, 2) == 0


def test_empty_calls_do_nothing():
    assert nnb.lib.nnb200_paged_append(*append_args(tokens=0, k=None, v=None)) == 0
    assert nnb.lib.nnb200_paged_attention(*attention_args(groups=0)) == 0
    assert nnb.lib.nnb200_paged_attention(*attention_args(size=0)) == 0
    assert nnb.lib.nnb200_beam_select(*select_args(groups=0)) == 0
    assert nnb.lib.nnb200_beam_reorder(*reorder_args(groups=0)) == 0
    assert nnb.lib.nnb200_beam_reorder(*reorder_args(beams=0)) == 0


def test_scratch_of_empty_calls():
    for groups, size in ((0, 0), (0, 100), (3, 0)):
        assert nnb.lib.nnb200_paged_attention_scratch_bytes(C.byref(kv()), groups, size, 4, 4, 2) < 1024
    assert nnb.lib.nnb200_beam_select_scratch_bytes(0, 4, 100, 8) < 1024


def test_one_layer_needs_no_stride():
    assert nnb.lib.nnb200_paged_append(*append_args(kv(layers=1, layer_stride=0), tokens=0)) == 0


def batch_cfg(**change):
    a = dict(vocab=72, d_model=128, heads=2, layers=2, d_ff=104, seq=64, batch=1, act=1, norm=1, pos=3, precision=0)
    a.update(change)
    return nnb.GptConfig(*a.values()).c_struct()


@pytest.mark.parametrize("change,seqs,rows", [({}, 0, 4), ({}, 1025, 4), ({}, 4, 0), ({}, 4, 65), (dict(d_model=24, heads=2), 4, 4), (dict(d_model=528, heads=2), 4, 4),
                                              (dict(d_model=130), 4, 4), (dict(seq=1 << 22), 1024, 1 << 22)])
def test_batch_refuses_shapes(change, seqs, rows):
    c = batch_cfg(**change)
    assert nnb.lib.nnb200_gpt_batch_workspace_bytes(C.byref(c), seqs, rows) == -1
    refused("nnb200_gpt_batch_begin", C.byref(c), P, P, seqs, rows, 10, None)
    refused("nnb200_gpt_batch_step", C.byref(c), P, P, P, P, seqs, rows, 10, 0, P, P, None)
    refused("nnb200_gpt_batch_reorder", C.byref(c), P, seqs, rows, P, None)


@pytest.mark.parametrize("heads,seqs", [(8192, 512), (70000, 1)])
def test_batch_refuses_more_heads_than_its_attention_takes(heads, seqs):
    """At once, and not in the first step behind a prompt."""
    c = batch_cfg(d_model=8 * heads, heads=heads, layers=1)
    assert nnb.lib.nnb200_gpt_batch_workspace_bytes(C.byref(c), seqs, 4) == -1
    refused("nnb200_gpt_batch_begin", C.byref(c), P, P, seqs, 4, 10, None)


def test_batch_refuses_arguments():
    c = batch_cfg()
    assert nnb.lib.nnb200_gpt_batch_workspace_bytes(C.byref(c), 4, 8) > 0
    for args in ((None, P, 4, 8, 10), (P, None, 4, 8, 10), (P, P + 128, 4, 8, 10), (P, P, 4, 8, 0), (P, P, 4, 8, 57), (P, P, 4, 8, -1)):
        refused("nnb200_gpt_batch_begin", C.byref(c), *args, None)
    good = dict(params=P, bf16=None, dec=P, ws=P, seqs=4, rows=8, prompt=10, step=0, tokens=P, logits=P)
    for change in (dict(params=None), dict(dec=None), dict(ws=None), dict(tokens=None), dict(logits=None), dict(params=P + 8), dict(ws=P + 16), dict(logits=P + 4), dict(step=-1),
                   dict(step=8), dict(prompt=0), dict(prompt=57)):
        refused("nnb200_gpt_batch_step", C.byref(c), *{**good, **change}.values(), None)
    refused("nnb200_gpt_batch_step", C.byref(batch_cfg(precision=1)), *good.values(), None)
    refused("nnb200_gpt_batch_reorder", C.byref(c), None, 4, 8, P, None)
    refused("nnb200_gpt_batch_reorder", C.byref(c), P, 4, 8, None, None)
