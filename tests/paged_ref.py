"""Plain 64-bit numpy forms of the batched-decoding operators (nnb200_paged_append, nnb200_paged_attention, nnb200_beam_select,
nnb200_beam_reorder), written row by row from their definitions, and the error bounds of their 32-bit kernels."""
import numpy as np

U = 2.0 ** -24                      # half a step of fp32
HALF_STEP = {0: 2.0 ** -24, 1: 2.0 ** -8}


def append(k_pages, v_pages, q, k, v, seq_of, row_of, table, rope, rope_pos, page_size):
    """k_pages, v_pages (pages, kv_heads, page_size, dk) float64, changed in place; q (n, heads, dk) or None, k, v (n, kv_heads, dk).
    Returns the rotated q, NaN rows for tokens left out."""
    pages, dk = k_pages.shape[0], k.shape[-1]
    out = None if q is None else np.full(q.shape, np.nan)
    for i in range(k.shape[0]):
        s, r = (i if seq_of is None else seq_of[i]), row_of[i]
        if not (0 <= s < table.shape[0]) or r < 0 or r // page_size >= table.shape[1]:
            continue
        p, pos = table[s, r // page_size], (r if rope_pos is None else rope_pos[i])
        if not 0 <= p < pages or (rope is not None and not 0 <= pos < rope.shape[1]):
            continue

        def turn(x):
            if rope is None:
                return x
            c, n, a, b = rope[0, pos], rope[1, pos], x[:, :dk // 2], x[:, dk // 2:]
            return np.concatenate([a * c - b * n, b * c + a * n], axis=1)
        k_pages[p, :, r % page_size] = turn(k[i])
        v_pages[p, :, r % page_size] = v[i]
        if q is not None:
            out[i] = turn(q[i])
    return out


def rows_of(pool, table, count, page_size):
    """(kv_heads, rows, dk) of the first `count` rows of a page table row, and which of them lie in pages that are there."""
    count = int(min(max(count, 0), len(table) * page_size))
    at = np.arange(count)
    page = np.asarray(table)[at // page_size] if count else np.zeros(0, np.int64)
    there = (page >= 0) & (page < pool.shape[0])
    got = np.zeros((pool.shape[1], count, pool.shape[3]))
    got[:, there] = pool[page[there], :, at[there] % page_size].transpose(1, 0, 2)
    return got, there


def attention(q, k_pages, v_pages, prefix_table, prefix_len, table, seq_len, size, alibi, dtype):
    """q (n, heads, dk), pools (pages, kv_heads, page_size, dk), float64.  Returns out, lse and bounds of their errors for a kernel
    that accumulates in fp32 (every sum of n terms off by n half steps), rounds weights and result to the type."""
    n, heads, dk = q.shape
    hk, ps = k_pages.shape[1], k_pages.shape[2]
    m = heads // hk
    out, lse = np.zeros(q.shape), np.full((n, heads), -np.inf)
    tol, tol_lse = np.zeros(q.shape), np.zeros((n, heads))
    for i in range(n):
        g = i // size
        if seq_len[i] < 0:
            continue
        kp, tp = rows_of(k_pages, prefix_table[g], prefix_len[g], ps) if prefix_table.shape[1] else (np.zeros((hk, 0, dk)), np.zeros(0, bool))
        ko, to = rows_of(k_pages, table[i], seq_len[i], ps) if table.shape[1] else (np.zeros((hk, 0, dk)), np.zeros(0, bool))
        vp = rows_of(v_pages, prefix_table[g], prefix_len[g], ps)[0] if prefix_table.shape[1] else kp
        vo = rows_of(v_pages, table[i], seq_len[i], ps)[0] if table.shape[1] else ko
        k, v, there = np.concatenate([kp, ko], 1), np.concatenate([vp, vo], 1), np.concatenate([tp, to])
        total = k.shape[1]
        if not there.any():
            continue
        back = np.arange(total - 1, -1, -1, dtype=np.float64)[there]
        k, v = k[:, there], v[:, there]
        for h in range(heads):
            slope = 2.0 ** (-8.0 * h / heads) if alibi else 0.0
            x = k[h // m] @ q[i, h] / np.sqrt(dk) - slope * back
            with np.errstate(invalid="ignore"):
                top = x.max()
                e = np.exp(x - (top if np.isfinite(top) or np.isnan(top) or top > 0 else 0.0))
            if e.sum() == 0.0:
                continue
            p = e / e.sum()
            out[i, h], lse[i, h] = p @ v[h // m], top + np.log(e.sum())
            # a score: dk products summed, scaled, the bias subtracted (slope, distance and product rounded); an exponential: 4 steps
            ds = np.max(U * ((dk + 3) * (np.abs(k[h // m]) @ np.abs(q[i, h])) / np.sqrt(dk) + 4 * slope * back + 2 * np.abs(x))) + 8 * U
            each = 2 * ds + 2 * (total + 40) * U + (HALF_STEP[1] if dtype else 0.0)
            tol[i, h] = each * (p @ np.abs(v[h // m])) + HALF_STEP[dtype] * np.abs(out[i, h]) + 1e-37
            tol_lse[i, h] = ds + (total + 40) * U + 2 * U * abs(lse[i, h])
    return out, lse, tol, tol_lse


def select(logits, scores, ended, eos, n):
    """logits (groups, beams, vocab), scores (groups, beams) float64.  Lists per group of (parent, token, score, ended), in 64 bits."""
    result = []
    for g in range(logits.shape[0]):
        cand = []
        for b in range(logits.shape[1]):
            if ended is not None and ended[g, b]:
                if scores[g, b] > -np.inf:
                    cand.append((-scores[g, b], b, eos))
                continue
            x = logits[g, b]
            if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all() or not scores[g, b] > -np.inf:
                continue
            top = x.max()
            norm = top + np.log(np.exp(x - top).sum())
            value = scores[g, b] + (x - norm)
            for t in np.argsort(-value, kind="stable")[:n]:
                if value[t] > -np.inf:
                    cand.append((-value[t], b, int(t)))
        cand.sort()
        row = [(b, t, -s, int(bool(ended is not None and ended[g, b]) or t == eos)) for s, b, t in cand[:n]]
        result.append(row + [(-1, -1, -np.inf, 0)] * (n - len(row)))
    return result


def reorder(k_pages, v_pages, parent, length, table, spare, beams):
    """k_pages, v_pages (layers, pages, kv_heads, page_size, dk), changed in place.  Returns length, table and spare after it."""
    n, ps = len(length), k_pages.shape[3]
    new_len, new_table, new_spare = np.zeros_like(length), table.copy(), spare.copy()
    old_k, old_v = k_pages.copy(), v_pages.copy()
    for i in range(n):
        p = i // beams * beams + parent[i] if 0 <= parent[i] < beams else i
        new_len[i] = length[p]
        rows = min(max(int(length[p]), 0), table.shape[1] * ps)
        full, rest = rows // ps, rows % ps
        new_table[i, :full] = table[p, :full]
        if rest:
            new_table[i, full], new_spare[i] = spare[i], table[i, full]
            src, dst = table[p, full], spare[i]
            if 0 <= src < k_pages.shape[1] and 0 <= dst < k_pages.shape[1]:
                k_pages[:, dst, :, :rest], v_pages[:, dst, :, :rest] = old_k[:, src, :, :rest], old_v[:, src, :, :rest]
    return new_len, new_table, new_spare
