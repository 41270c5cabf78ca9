"""Performance cases of the operators of batched decoding: several continuations of a prompt over a paged key/value cache.

Operators
  append     new tokens' keys and values into the cache's pages, keys and queries rotated to their positions on the way
  attention  one new query per sequence over a prefix that the sequences of a group share, then over the sequence's own rows
  select     the best continuations of each group over its beams and the vocabulary
  reorder    the states of the chosen beams: whole pages through the page table, the last one, partly filled, copied

A pool of pages is (pages, kv_heads, page_size, head_dim) for keys and the same for values; row t of a sequence is row
t % page_size of page table[t // page_size].

Model sizes are those of the repository's configurations and tests, or generic ones between them.
"""
import ctypes as C
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
CODES = {"fp32": 0, "bf16": 1}


def _append(name, dtype, src, heads, kv_heads, dk, page, seqs, longest, tokens, rope):
    c = dict(op="append", dtype=dtype, src=src, heads=heads, kv_heads=kv_heads, dk=dk, page=page, seqs=seqs, longest=longest, tokens=tokens, rope=rope)
    return dict(c, name=name) if name else c


def _attention(name, dtype, heads, kv_heads, dk, page, groups, size, prefix, longest, ragged, alibi):
    c = dict(op="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dk=dk, page=page, groups=groups, size=size, prefix=prefix, longest=longest,
             ragged=ragged, alibi=alibi)
    return dict(c, name=name) if name else c


def _select(name, dtype, groups, beams, vocab, n, ended):
    c = dict(op="select", dtype=dtype, groups=groups, beams=beams, vocab=vocab, n=n, ended=ended)
    return dict(c, name=name) if name else c


def _reorder(name, dtype, layers, kv_heads, dk, page, groups, beams, length, capacity):
    c = dict(op="reorder", dtype=dtype, layers=layers, kv_heads=kv_heads, dk=dk, page=page, groups=groups, beams=beams, length=length, capacity=capacity)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of each of eight beams of the benchmark model, fp32 as decoding keeps it: pure latency
        _append("append_step", "fp32", "fp32", 12, 12, 64, 16, 8, 1024, 8, True),
        # a serving batch, grouped heads of 128, a long cache
        _append("append_batch", "bf16", "bf16", 32, 8, 128, 64, 192, 768, 192, True),
        # prompts of a few sequences at once, fp32 activations into a bf16 cache
        _append("append_prompts", "bf16", "fp32", 16, 16, 64, 32, 7, 2048, 8192, True),
        # four beams of the small model shortly behind a short prompt: pure latency
        _attention("attention_small", "fp32", 6, 6, 64, 16, 1, 4, 41, 16, False, False),
        # eight beams of the benchmark model late in its window
        _attention("attention_base", "fp32", 12, 12, 64, 16, 1, 8, 901, 100, False, True),
        # many prompts at once, beams of each; an odd page end everywhere
        _attention("attention_groups", "bf16", 16, 16, 64, 16, 16, 8, 2047, 253, True, False),
        # many answers behind one long system prompt
        _attention("attention_batch", "bf16", 16, 16, 64, 32, 1, 64, 8192, 512, True, False),
        # grouped heads of 128 behind a very long document, the largest call
        _attention("attention_long", "bf16", 32, 8, 128, 64, 1, 96, 32768, 1024, True, False),
        # the beams of the small model
        _select("select_small", "fp32", 1, 4, 4096, 4, False),
        # a serving batch with a large vocabulary, some beams already at their end
        _select("select_batch", "bf16", 64, 8, 32768, 16, True),
        # beams of the benchmark model
        _reorder("reorder_base", "fp32", 12, 12, 64, 16, 1, 8, 107, 256),
        # a serving batch of a larger model
        _reorder("reorder_batch", "bf16", 16, 8, 128, 32, 24, 8, 94, 128),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    group = rng.choice([1, 1, 1, 2, 3, 4, 8])
    return kv * group, kv, rng.choice([32, 64, 64, 64, 80, 96, 128, 128])


def draw(rng):
    """One more case of the same ranges: sizes over their logarithms, odd ones among them."""
    op = rng.choices(["append", "attention", "select", "reorder"], [20, 45, 20, 15])[0]
    dtype = rng.choice(["fp32", "bf16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    while True:
        heads, kv_heads, dk = _heads(rng)
        if op == "append":
            tokens = round(_log(rng, 1, 8192))
            seqs = tokens if tokens <= 256 and rng.random() < 0.7 else rng.randint(1, 16)
            longest = max(-(-tokens // seqs), round(_log(rng, 32, 2048)))
            c = _append(None, dtype, dtype if rng.random() < 0.7 else "fp32", heads, kv_heads, dk, page, seqs, longest, tokens, rng.random() < 0.8)
        elif op == "attention":
            groups = rng.choice([1, 1, 1, 2, 5, 16])
            size = round(_log(rng, 1, 96))
            prefix = round(_log(rng, 8, 32768)) if rng.random() < 0.9 else 0
            c = _attention(None, dtype, heads, kv_heads, dk, page, groups, size, prefix, round(_log(rng, 1, 1024)), rng.random() < 0.7, rng.random() < 0.25)
        elif op == "select":
            beams = rng.randint(1, 16)
            c = _select(None, dtype, round(_log(rng, 1, 64)), beams, round(_log(rng, 500, 65536)), beams * rng.choice([1, 2]), rng.random() < 0.5)
        else:
            beams = rng.randint(1, 16)
            capacity = round(_log(rng, 16, 256))
            c = _reorder(None, dtype, round(_log(rng, 1, 16)), kv_heads, dk, page, round(_log(rng, 1, 24)), beams, rng.randint(1, capacity), capacity)
        w = work(c)
        # the operator's own largest call bounds what it may cost, and the pool what a card holds beside it three times over
        most = {"append": 1.5e8, "attention": 3.2e8, "select": 3.3e7, "reorder": 7.5e8}[op]
        if w["bytes"] <= most and w["flops"] <= (4.8e10 if dtype == "bf16" else 1.6e10) and _pool_bytes(c) <= 2e9:
            return c


# ---------------------------------------------------------------------------------------------- inputs
def _size(dtype):
    return 4 if dtype == "fp32" else 2


def _pages(c):
    """(pages of a shared prefix, pages of a sequence's own rows, pages of the pool) of a case."""
    up = lambda n: -(-n // c["page"])  # noqa: E731
    if c["op"] == "append":
        return 0, up(c["longest"]), c["seqs"] * up(c["longest"]) + 3
    if c["op"] == "attention":
        return up(c["prefix"]), up(c["longest"]), c["groups"] * (up(c["prefix"]) + c["size"] * up(c["longest"])) + 3
    return 0, up(c["capacity"]), c["groups"] * c["beams"] * (up(c["capacity"]) + 1)


def _pool_bytes(c):
    if c["op"] == "select":
        return 0
    return 2 * _pages(c)[2] * c["kv_heads"] * c["page"] * c["dk"] * c.get("layers", 1) * _size(c["dtype"])


def _lengths(c, gen):
    """Prefix length of each group and own rows of each sequence, as whole numbers on the CPU.  Ragged: from one row up, one
    sequence in sixteen of a batch a padded one (no rows, nothing visible: length -1)."""
    n = c["groups"] * c["size"]
    if not c["ragged"]:
        return torch.full((c["groups"],), c["prefix"], dtype=torch.int32), torch.full((n,), c["longest"], dtype=torch.int32)
    low = max(1, c["prefix"] // 2) if c["prefix"] else 0
    prefix = torch.randint(low, c["prefix"] + 1, (c["groups"],), generator=gen, dtype=torch.int32)
    prefix[0] = c["prefix"]
    rows = torch.randint(1, c["longest"] + 1, (n,), generator=gen, dtype=torch.int32)
    rows[torch.arange(n) % 16 == 15] = -1
    return prefix, rows


def _work_lengths(c):
    """Mean sums of the same over their distribution: (prefix rows of all groups, own rows of all sequences, rows that queries see)."""
    n = c["groups"] * c["size"]
    if not c["ragged"]:
        return c["groups"] * c["prefix"], n * c["longest"], n * (c["prefix"] + c["longest"])
    mean = (max(1, c["prefix"] // 2) + c["prefix"]) / 2 if c["prefix"] else 0
    prefix = c["prefix"] + (c["groups"] - 1) * mean
    live = n - n // 16
    own_rows = live * (c["longest"] + 1) / 2
    return prefix, own_rows, live * prefix / c["groups"] + own_rows


def _pool(c, gen):
    shape = (c.get("layers", 1), _pages(c)[2], c["kv_heads"], c["page"], c["dk"])
    make = lambda: torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32 if c["dtype"] == "fp32" else torch.bfloat16)  # noqa: E731
    return make(), make()


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    t = TYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "append":
        s["k_pages"], s["v_pages"] = _pool(c, gen)
        _, per, pages = _pages(c)
        s["table"] = torch.randperm(pages, generator=cpu)[:c["seqs"] * per].to(torch.int32).view(c["seqs"], per).cuda()
        # each sequence gets a run of new tokens behind a random number of rows it has
        share = torch.tensor([c["tokens"] // c["seqs"] + (i < c["tokens"] % c["seqs"]) for i in range(c["seqs"])])
        seq = torch.repeat_interleave(torch.arange(c["seqs"]), share)
        start = (torch.rand(c["seqs"], generator=cpu) * (c["longest"] - share + 1)).long()
        first = torch.cumsum(share, 0) - share
        s["seq_of"] = seq.to(torch.int32).cuda()
        s["row_of"] = (start[seq] + torch.arange(c["tokens"]) - first[seq]).to(torch.int32).cuda()
        width = (c["heads"] + 2 * c["kv_heads"]) * c["dk"]
        s["qkv"] = torch.randn((c["tokens"], width), device="cuda", generator=gen).to(TYPES[c["src"]])
        s["q_out"] = torch.empty((c["tokens"], c["heads"] * c["dk"]), device="cuda", dtype=t)
        half = c["dk"] // 2
        angle = torch.arange(c["longest"], dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(half, dtype=torch.float64) * 2 / c["dk"])
        s["rope"] = torch.cat([angle.cos().flatten(), angle.sin().flatten()]).float().cuda() if c["rope"] else None
    elif c["op"] == "attention":
        s["k_pages"], s["v_pages"] = _pool(c, gen)
        shared, per, pages = _pages(c)
        n = c["groups"] * c["size"]
        order = torch.randperm(pages, generator=cpu).to(torch.int32)
        s["prefix_table"] = order[:c["groups"] * shared].view(c["groups"], shared).cuda()
        s["table"] = order[c["groups"] * shared:c["groups"] * shared + n * per].view(n, per).cuda()
        prefix, rows = _lengths(c, cpu)
        s["prefix_len"], s["len"] = prefix.cuda(), rows.cuda()
        s["q"] = (2.0 * torch.randn((n, c["heads"] * c["dk"]), device="cuda", generator=gen)).to(t)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((n, c["heads"]), device="cuda")
    elif c["op"] == "select":
        rows = c["groups"] * c["beams"]
        s["logits"] = (3.0 * torch.randn((rows, c["vocab"]), device="cuda", generator=gen)).to(t)
        s["scores"] = -torch.sort(40.0 * torch.rand((c["groups"], c["beams"]), device="cuda", generator=gen), dim=1).values.flatten() * 0.1 - 5.0
        s["eos"] = 2
        s["ended"] = (torch.rand(rows, device="cuda", generator=gen) < 0.1).to(torch.int32) if c["ended"] else torch.zeros(rows, dtype=torch.int32, device="cuda")
        shape = (c["groups"], c["n"])
        s["parent"], s["token"], s["ended_out"] = (torch.empty(shape, dtype=torch.int32, device="cuda") for _ in "pte")
        s["scores_out"] = torch.empty(shape, device="cuda")
    else:
        s["k_pages"], s["v_pages"] = _pool(c, gen)
        _, per, pages = _pages(c)
        n = c["groups"] * c["beams"]
        order = torch.randperm(pages, generator=cpu).to(torch.int32)
        s["table"], s["spare"] = order[:n * per].view(n, per).cuda(), order[n * per:n * per + n].cuda()
        s["len"] = torch.full((n,), c["length"], dtype=torch.int32, device="cuda")
        s["parent"] = torch.randint(0, c["beams"], (n,), generator=cpu, dtype=torch.int32).cuda()
        s["table_out"], s["spare_out"], s["len_out"] = torch.empty_like(s["table"]), torch.empty_like(s["spare"]), torch.empty_like(s["len"])
    s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _rotated(x, rope, pos, dk):
    """(tokens, heads, dk) fp32 rotated by halves to the positions; rope: cosines (rows, dk / 2), then sines."""
    table = rope.view(2, -1, dk // 2)
    cos, sin = table[0][pos][:, None, :], table[1][pos][:, None, :]
    a, b = x[..., :dk // 2], x[..., dk // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_append(c, s):
    x = s["qkv"].float()
    n, h, hk, dk = c["tokens"], c["heads"], c["kv_heads"], c["dk"]
    q, k, v = x[:, :h * dk].reshape(n, h, dk), x[:, h * dk:(h + hk) * dk].reshape(n, hk, dk), x[:, (h + hk) * dk:].reshape(n, hk, dk)
    row = s["row_of"].long()
    if s["rope"] is not None:
        q, k = _rotated(q, s["rope"], row, dk), _rotated(k, s["rope"], row, dk)
    page = s["table"][s["seq_of"].long(), row // c["page"]].long()
    s["k_pages"][0][page, :, row % c["page"]] = k.to(s["k_pages"].dtype)
    s["v_pages"][0][page, :, row % c["page"]] = v.to(s["v_pages"].dtype)
    s["q_out"].copy_(q.reshape(n, h * dk))
    return s["q_out"], s["k_pages"], s["v_pages"]


def _rows(pool, table):
    """(sequences, kv_heads, rows, dk) fp32 of the pages in a table."""
    got = pool[0][table.long()].float()
    n, p, h, r, d = got.shape
    return got.permute(0, 2, 1, 3, 4).reshape(n, h, p * r, d)


def _plain_attention(c, s):
    g, b, h, hk, dk = c["groups"], c["size"], c["heads"], c["kv_heads"], c["dk"]
    m = h // hk
    q = s["q"].float().view(g, b, hk, m, dk)
    dev = q.device
    prefix, own_len = s["prefix_len"].view(g, 1), s["len"].view(g, b)
    live = own_len >= 0
    kp, vp = _rows(s["k_pages"], s["prefix_table"]), _rows(s["v_pages"], s["prefix_table"])                # (g, hk, P, dk)
    ko, vo = (_rows(s[x], s["table"]).view(g, b, hk, -1, dk) for x in ("k_pages", "v_pages"))              # (g, b, hk, L, dk)
    n_p, n_o = kp.shape[2], ko.shape[3]
    scores = torch.cat([torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(g, hk, b * m, dk), kp.transpose(-1, -2)).view(g, hk, b, m, n_p).permute(0, 2, 1, 3, 4),
                        torch.matmul(q, ko.transpose(-1, -2))], dim=-1) * (1.0 / math.sqrt(dk))            # (g, b, hk, m, P + L)
    at_p, at_o = torch.arange(n_p, device=dev), torch.arange(n_o, device=dev)
    seen = torch.cat([(at_p < prefix[..., None]).expand(g, b, n_p) & live[..., None], at_o < own_len[..., None]], dim=-1)
    if c["alibi"]:
        slope = torch.exp2(-8.0 * torch.arange(h, device=dev, dtype=torch.float32) / h).view(hk, m)
        place = torch.cat([at_p.expand(g, n_p), prefix + at_o], dim=-1).view(g, 1, -1)
        back = (prefix + own_len - 1)[..., None] - place
        scores = scores - slope[:, :, None] * back[:, :, None, None, :]
    scores = scores.masked_fill(~seen[:, :, None, None, :], -math.inf)
    top = scores.max(dim=-1, keepdim=True).values
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    shared = torch.matmul(p[..., :n_p].permute(0, 2, 1, 3, 4).reshape(g, hk, b * m, n_p), vp).view(g, hk, b, m, dk).permute(0, 2, 1, 3, 4)
    s["out"].copy_((shared + torch.matmul(p[..., n_p:], vo)).reshape(g * b, h * dk))
    s["lse"].copy_((top + torch.log(total)).reshape(g * b, h))
    return s["out"], s["lse"]


def _plain_select(c, s):
    g, b, v, n = c["groups"], c["beams"], c["vocab"], c["n"]
    x = s["logits"].double().view(g, b, v)
    top = x.max(dim=-1, keepdim=True).values
    value = s["scores"].double().view(g, b, 1) + (x - (top + torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))))
    ended = s["ended"].view(g, b, 1) != 0
    only = torch.where(torch.arange(v, device=x.device) == s["eos"], s["scores"].double().view(g, b, 1), -math.inf)
    value, at = torch.sort(torch.where(ended, only, value).view(g, b * v), dim=-1, descending=True, stable=True)
    value, at = value[:, :n], at[:, :n]
    gone = value == -math.inf
    parent, token = torch.where(gone, -1, at // v), torch.where(gone, -1, at % v)
    s["parent"].copy_(parent)
    s["token"].copy_(token)
    s["scores_out"].copy_(value)
    s["ended_out"].copy_(torch.where(gone, False, torch.gather(ended.view(g, b), 1, parent.clamp(min=0)) | (token == s["eos"])))
    return s["parent"], s["token"], s["scores_out"], s["ended_out"]


def _plain_reorder(c, s):
    g, b, page = c["groups"], c["beams"], c["page"]
    from_ = (torch.arange(g, device="cuda")[:, None] * b + s["parent"].view(g, b).long()).flatten()
    length = s["len"][from_]
    full, rest = (length // page)[:, None], (length % page)[:, None]
    at = torch.arange(s["table"].shape[1], device="cuda")
    partly = (at == full) & (rest > 0)
    last = full.long().clamp(max=s["table"].shape[1] - 1)
    s["table_out"].copy_(torch.where(at < full, s["table"][from_], torch.where(partly, s["spare"][:, None], s["table"])))
    s["spare_out"].copy_(torch.where(rest[:, 0] > 0, torch.gather(s["table"], 1, last)[:, 0], s["spare"]))
    s["len_out"].copy_(length)
    src, dst = torch.gather(s["table"][from_], 1, last)[:, 0].long(), s["spare"].long()
    copied = (torch.arange(page, device="cuda") < rest)[None, :, None, :, None]
    s["k_pages"][:, dst] = torch.where(copied, s["k_pages"][:, src], s["k_pages"][:, dst])
    s["v_pages"][:, dst] = torch.where(copied, s["v_pages"][:, src], s["v_pages"][:, dst])
    return s["table_out"], s["spare_out"], s["len_out"], s["k_pages"], s["v_pages"]


# ---------------------------------------------------------------------------------------------- the framework's operators
def _handle(nnb, c, s):
    """The cache's description, and the workspace, as a decoding program makes them once."""
    if c["op"] != "select":
        layers = c.get("layers", 1)
        s["kv"] = C.byref(nnb.PagedKv(s["at"]["k_pages"], s["at"]["v_pages"], s["k_pages"][0].numel(), layers, s["k_pages"].shape[1], c["page"], c["kv_heads"],
                                      c["dk"], CODES[c["dtype"]]))
    size = 0
    if c["op"] == "attention":
        size = nnb.call("nnb200_paged_attention_scratch_bytes", s["kv"], c["groups"], c["size"], c["heads"], s["prefix_table"].shape[1], s["table"].shape[1])
    elif c["op"] == "select":
        size = nnb.call("nnb200_beam_select_scratch_bytes", c["groups"], c["beams"], c["vocab"], c["n"])
    s["scratch"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    s["nnb"] = nnb


def _own(c, s):
    if "nnb" not in s:
        import __graft_entry__ as entry
        _handle(entry.load_package(), c, s)
    call, at, scratch = s["nnb"].call, s["at"], s["scratch"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        es, dk, h, hk = _size(c["src"]), c["dk"], c["heads"], c["kv_heads"]
        ld = (h + 2 * hk) * dk
        call("nnb200_paged_append", s["kv"], 0, at["qkv"], ld, at["q_out"], h * dk, at["qkv"] + h * dk * es, at["qkv"] + (h + hk) * dk * es, ld, CODES[c["src"]],
             c["tokens"], h, at["seq_of"], at["row_of"], at["table"], c["seqs"], s["table"].shape[1], at.get("rope"), c["longest"] if c["rope"] else 0, None, stream)
        return s["q_out"], s["k_pages"], s["v_pages"]
    if c["op"] == "attention":
        ld = c["heads"] * c["dk"]
        call("nnb200_paged_attention", s["kv"], 0, at["q"], ld, at["out"], ld, at["lse"], at["prefix_table"], s["prefix_table"].shape[1], at["prefix_len"], at["table"],
             s["table"].shape[1], at["len"], c["groups"], c["size"], c["heads"], 1 if c["alibi"] else 0, scratch.data_ptr(), scratch.numel(), stream)
        return s["out"], s["lse"]
    if c["op"] == "select":
        call("nnb200_beam_select", at["logits"], c["vocab"], CODES[c["dtype"]], c["groups"], c["beams"], c["vocab"], at["scores"], at["ended"], s["eos"], c["n"],
             at["parent"], at["token"], at["scores_out"], at["ended_out"], scratch.data_ptr(), scratch.numel(), stream)
        return s["parent"], s["token"], s["scores_out"], s["ended_out"]
    call("nnb200_beam_reorder", s["kv"], c["groups"], c["beams"], at["parent"], at["len"], at["table"], at["spare"], at["len_out"], at["table_out"], at["spare_out"],
         s["table"].shape[1], stream)
    return s["table_out"], s["spare_out"], s["len_out"], s["k_pages"], s["v_pages"]


def run(s):
    c = s["case"]
    if own:
        return _own(c, s)
    return {"append": _plain_append, "attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder}[c["op"]](c, s)


# ---------------------------------------------------------------------------------------------- work
def work(c):
    es = _size(c.get("dtype"))
    if c["op"] == "append":
        wide = (c["heads"] + 2 * c["kv_heads"]) * c["dk"]
        turned = (c["heads"] + c["kv_heads"]) * c["dk"] if c["rope"] else 0
        table = 4 * c["dk"] * min(c["longest"], c["tokens"]) if c["rope"] else 0
        return {"bytes": c["tokens"] * (wide * (_size(c["src"]) + es) + 12) + table, "flops": 3 * c["tokens"] * turned}
    if c["op"] == "attention":
        prefix, rows, seen = _work_lengths(c)
        io = 2 * c["groups"] * c["size"] * c["heads"] * c["dk"] * es
        return {"bytes": 2 * (prefix + rows) * c["kv_heads"] * c["dk"] * es + io, "flops": 4 * seen * c["heads"] * c["dk"]}
    if c["op"] == "select":
        rows = c["groups"] * c["beams"]
        return {"bytes": rows * (c["vocab"] * es + 8) + c["groups"] * c["n"] * 16, "flops": 3 * rows * c["vocab"]}
    rest = c["length"] % c["page"]
    n = c["groups"] * c["beams"]
    return {"bytes": 4 * n * rest * c["layers"] * c["kv_heads"] * c["dk"] * es + 8 * n * (_pages(c)[1] + 4), "flops": 0}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_attention(c, s):
    g, b, h, hk, dk, page = c["groups"], c["size"], c["heads"], c["kv_heads"], c["dk"], c["page"]
    m = h // hk
    k, v = s["k_pages"][0], s["v_pages"][0]
    out = torch.zeros((g * b, h, dk), dtype=torch.float64, device="cuda")
    lse = torch.full((g * b, h), -math.inf, dtype=torch.float64, device="cuda")
    slope = 2.0 ** (-8.0 * torch.arange(h, dtype=torch.float64, device="cuda") / h) if c["alibi"] else torch.zeros(h, dtype=torch.float64, device="cuda")
    prefix, rows = s["prefix_len"].tolist(), s["len"].tolist()

    def keys(pool, table, count):
        """(hk, count, dk) of one table row."""
        got = pool[table[:-(-count // page)].long()].double() if count > 0 else pool[:0].double()
        return got.transpose(0, 1).reshape(hk, -1, dk)[:, :max(count, 0)]

    for j in range(g):
        kp, vp = keys(k, s["prefix_table"][j], prefix[j]), keys(v, s["prefix_table"][j], prefix[j])
        for i in range(j * b, (j + 1) * b):
            if rows[i] < 0 or prefix[j] + rows[i] == 0:
                continue
            q = s["q"][i].double().view(hk, m, dk)
            far = torch.arange(prefix[j] + rows[i] - 1, -1, -1, dtype=torch.float64, device="cuda")
            ko, vo = keys(k, s["table"][i], rows[i]), keys(v, s["table"][i], rows[i])
            x = torch.cat([q @ kp.transpose(1, 2), q @ ko.transpose(1, 2)], dim=2) / math.sqrt(dk) - slope.view(hk, m, 1) * far
            lse[i] = torch.logsumexp(x, dim=2).flatten()
            p = torch.softmax(x, dim=2)
            out[i] = (p[..., :prefix[j]] @ vp + p[..., prefix[j]:] @ vo).reshape(h, dk)
    return out.view(g * b, h * dk), lse


def exact(c, seed):
    if c["op"] == "attention":
        return _exact_attention(c, prepare(c, seed)) if work(c)["flops"] <= 2e11 else None
    if c["op"] == "append":
        s = prepare(c, seed)
        k, v = s["k_pages"].double(), s["v_pages"].double()
        h, hk, half = c["heads"], c["kv_heads"], c["dk"] // 2
        x = s["qkv"].double().view(c["tokens"], h + 2 * hk, 2, half)
        row = s["row_of"].long()
        turn = torch.complex(s["rope"][:c["longest"] * half], s["rope"][c["longest"] * half:]).to(torch.complex128).view(-1, half)[row] if c["rope"] else torch.ones((), dtype=torch.complex128, device="cuda")
        z = torch.complex(x[:, :h + hk, 0], x[:, :h + hk, 1]) * (turn[:, None] if c["rope"] else turn)
        z = torch.stack([z.real, z.imag], dim=2).reshape(c["tokens"], h + hk, c["dk"])
        page = s["table"].long()[s["seq_of"].long(), torch.div(row, c["page"], rounding_mode="floor")]
        k[0, page, :, row % c["page"]] = z[:, h:]
        v[0, page, :, row % c["page"]] = x[:, h + hk:].reshape(c["tokens"], hk, c["dk"])
        return z[:, :h].reshape(c["tokens"], -1), k, v
    if c["op"] == "select":
        s = prepare(c, seed)
        g, b, v, n = c["groups"], c["beams"], c["vocab"], c["n"]
        x = torch.log_softmax(s["logits"].double(), dim=1) + s["scores"].double()[:, None]
        done = s["ended"].bool()
        x[done] = -math.inf
        x[done, s["eos"]] = s["scores"].double()[done]
        return None, None, torch.topk(x.view(g, b * v), n, dim=1).values, None
    s = prepare(c, seed)
    k, v = s["k_pages"].double(), s["v_pages"].double()
    rest = c["length"] % c["page"]
    if rest:
        table, parent, spare, b = s["table"].tolist(), s["parent"].tolist(), s["spare"].tolist(), c["beams"]
        for i in range(c["groups"] * b):
            page = table[i // b * b + parent[i]][c["length"] // c["page"]]
            k[:, spare[i], :, :rest] = s["k_pages"][:, page, :, :rest].double()
            v[:, spare[i], :, :rest] = s["v_pages"][:, page, :, :rest].double()
    return None, None, None, k, v
