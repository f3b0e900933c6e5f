"""Plain 64-bit implementations of the operators of a decode step over trees of drafted
tokens, written from their definitions, one sequence, row and head at a time."""
from __future__ import annotations

import torch


def mask_words(visible: list[list[set[int]]], words: int) -> torch.Tensor:
    """(total_q, words) int64 of the nodes that each row sees (per sequence, per row)."""
    rows = []
    for seq in visible:
        for sees in seq:
            v = sum(1 << j for j in sees if j < 64 * words)
            ws = [(v >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
            rows.append([w - (1 << 64) if w >> 63 else w for w in ws])
    return torch.tensor(rows, dtype=torch.int64).reshape(len(rows), words)


def paged_tree_ref(q, k_cache, v_cache, block_tables, context_lens, cu, visible, scale, k_scale=None,
                   v_scale=None):
    """(out, mag, mags): float64 attention; mag = sum_t w_t |v_t| per output, the size that
    relative errors of the weights act on; mags = max_t scale * sum_d |q_d k_d| per
    (row, head), the size that errors of the scores act on. Rows that see nothing are 0;
    rows of no sequence are NaN in `out`. Caches are (NB, BS, KVH, D); scales are one value
    or (NB, BS, KVH)."""
    NB, BS, KVH, D = k_cache.shape
    H = q.shape[1]
    G = H // KVH
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    mags = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    width = block_tables.shape[1]
    for b in range(len(visible)):
        q0, n = int(cu[b]), int(cu[b + 1]) - int(cu[b])
        ctx = int(context_lens[b])
        prefix = max(ctx - n, 0)
        tokens, page = [], []
        for t in range(min(max(ctx, 0), width * BS)):
            pg = int(block_tables[b, t // BS])
            if 0 <= pg < NB:
                tokens.append(t)
                page.append(pg)
        tt = torch.tensor(tokens, dtype=torch.int64, device=q.device)
        pp = torch.tensor(page, dtype=torch.int64, device=q.device)
        for i in range(n):
            on = torch.tensor([t < prefix or (t - prefix) in visible[b][i] for t in tokens],
                              dtype=torch.bool, device=q.device)
            row = q0 + i
            if not bool(on.any()):
                out[row] = 0.0
                continue
            t, pg = tt[on], pp[on]
            k, v = k_cache[pg, t % BS].double(), v_cache[pg, t % BS].double()  # (T, KVH, D)
            if k_scale is not None:
                ks = k_scale.double() if k_scale.numel() == 1 else k_scale[pg, t % BS].double()[..., None]
                vs = v_scale.double() if v_scale.numel() == 1 else v_scale[pg, t % BS].double()[..., None]
                k, v = k * ks, v * vs
            qq = q[row].double().view(KVH, G, D)
            s = torch.einsum("hgd,thd->hgt", qq, k) * scale
            w = torch.softmax(s, -1)
            out[row] = torch.einsum("hgt,thd->hgd", w, v).reshape(H, D)
            mag[row] = torch.einsum("hgt,thd->hgd", w, v.abs()).reshape(H, D)
            mags[row] = (torch.einsum("hgd,thd->hgt", qq.abs(), k.abs()) * abs(scale)).amax(-1).reshape(H)
    return out, mag, mags


def tree_metadata_ref(parents, cu, prefix, tables, block_size, words):
    """(slots, lens, positions, visible): lists, a slot per row, visible as node sets."""
    slots, lens, positions, visible = [], [], [], []
    for b in range(len(prefix)):
        n = cu[b + 1] - cu[b]
        lens.append(prefix[b] + n)
        rows = []
        for j in range(n):
            sees, a = set(), j
            while a >= 0:
                sees.add(a)
                p = parents[cu[b] + a]
                a = p if -1 <= p < a else -1
            t = prefix[b] + j
            page = tables[b][t // block_size] if t // block_size < len(tables[b]) else -1
            ok = j < 64 * words
            slots.append(page * block_size + t % block_size if ok and page >= 0 else -1)
            positions.append(prefix[b] + (len(sees) - 1 if ok else 0))
            rows.append(sees if ok else set())
        visible.append(rows)
    return slots, lens, positions, visible


def tree_accept_ref(draft, target, parents, cu, prefix, tables, block_size, max_path):
    """(count, nodes, tokens, lens, src, dst) as lists."""
    def slot(b, t):
        page = tables[b][t // block_size] if t // block_size < len(tables[b]) else -1
        return page * block_size + t % block_size if page >= 0 else -1

    out = ([], [], [], [], [], [])
    for b in range(len(prefix)):
        n = cu[b + 1] - cu[b]
        path = [0] if n else []
        while path and len(path) < max_path:
            c = path[-1]
            nxt = [d for d in range(c + 1, n) if parents[cu[b] + d] == c and draft[cu[b] + d] == target[cu[b] + c]]
            if not nxt:
                break
            path.append(nxt[0])
        pad = [-1] * (max_path - len(path))
        out[0].append(len(path))
        out[1].append(path + pad)
        out[2].append([target[cu[b] + c] for c in path] + pad)
        out[3].append(prefix[b] + len(path))
        out[4].append([slot(b, prefix[b] + c) if c != k else -1 for k, c in enumerate(path)] + pad)
        out[5].append([slot(b, prefix[b] + k) if c != k else -1 for k, c in enumerate(path)] + pad)
    return out
