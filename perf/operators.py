"""Cases and plain forms of the operators of a speculative decoding step over the paged KV cache.

A step with a tree of drafted tokens runs, per batch: `tree_metadata` (slots, positions,
lengths and ancestor masks of the drafted nodes), the model with `paged_attention_tree` in
each layer, `tree_accept` (the path of nodes that the target model agrees with) and
`move_kv_rows` (the accepted rows moved to the end of the sequence's cached prefix).
`copy_kv_pages` is what a forked sequence or a compacted cache needs of the GPU.

`run` computes an operator in its plain form (elementary torch operations in 32 bits), or,
where `own` is true, through the framework's entry points. Lengths and node counts come
from the case (`lens_seed`), everything else from the seed given to `prepare`.
"""
import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCAB = 151936


def _framework():
    """The framework's modules (the package's directory name holds a hyphen)."""
    return (importlib.import_module("mini-kvllm_b200.layers.attention"),
            importlib.import_module("mini-kvllm_b200.engine.kv_cache"))


# ------------------------------------------------------------------------------ cases
def listed():
    attn = {"op": "attention", "head_dim": 128, "kv_heads": 8}
    shape = {"layers": 28, "kv_heads": 8, "head_dim": 128}
    return [
        # one user's stream on the 16 / 8 head model: a shallow tree, a short prompt; latency
        dict(attn, name="attention_one_stream", dtype="bf16", cache="auto", heads=16, batch=1, block_size=16,
             ctx_min=411, ctx_max=411, nodes_min=8, nodes_max=8, lens_seed=1),
        # the 32 / 8 head model's serving batch with contexts of 1k to 8k, trees of 8 to 32 nodes
        dict(attn, name="attention_batch", dtype="bf16", cache="auto", heads=32, batch=48, block_size=256,
             ctx_min=1024, ctx_max=8192, nodes_min=8, nodes_max=32, lens_seed=2),
        # long documents in an e4m3 cache with per-tensor scales, contexts of 32k, full trees
        dict(attn, name="attention_long_fp8", dtype="bf16", cache="fp8_per_tensor", heads=32, batch=12,
             block_size=256, ctx_min=32768, ctx_max=32768, nodes_min=32, nodes_max=32, lens_seed=3),
        # odd sizes: int8 rows with their own scales, a ragged batch with single-token trees in it
        dict(attn, name="attention_odd_int8", dtype="fp16", cache="int8_per_token_head", heads=40, batch=19,
             block_size=16, ctx_min=1, ctx_max=5003, nodes_min=1, nodes_max=29, lens_seed=4),
        # the nodes of one stream's tree, and of a full batch of ragged trees
        dict(name="metadata_one_stream", op="metadata", batch=1, block_size=16, ctx_min=411, ctx_max=411,
             nodes_min=8, nodes_max=8, lens_seed=5),
        dict(name="metadata_batch", op="metadata", batch=256, block_size=256, ctx_min=1024, ctx_max=8192,
             nodes_min=17, nodes_max=96, lens_seed=6),
        # verification of one stream's tree, and of a full batch of ragged trees
        dict(name="accept_one_stream", op="accept", batch=1, block_size=16, ctx_min=411, ctx_max=411,
             nodes_min=8, nodes_max=8, max_path=6, lens_seed=7),
        dict(name="accept_batch", op="accept", batch=256, block_size=256, ctx_min=1024, ctx_max=8192,
             nodes_min=17, nodes_max=96, max_path=9, lens_seed=8),
        # one request forked into three further samples: its last, partly filled page is copied
        dict(shape, name="copy_fork", op="copy", dtype="bf16", block_size=16, pages=64, pairs=3),
        # a fragmented cache compacted: live pages at its end moved into holes at its start
        dict(shape, name="copy_compact", op="copy", dtype="bf16", block_size=16, pages=701, pairs=233),
        # the accepted rows of one stream, and of a full batch
        dict(shape, name="move_one_stream", op="move", dtype="bf16", block_size=16, batch=1, nodes=16, max_path=5,
             lens_seed=9),
        dict(shape, name="move_batch", op="move", dtype="bf16", block_size=16, batch=253, nodes=33, max_path=8,
             lens_seed=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "metadata", "accept", "copy", "move"])
    seed = rng.randrange(1 << 30)
    if op == "attention":
        cache = rng.choice(["auto", "auto", "fp8_per_tensor", "fp8_per_token_head", "int8_per_token_head"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        kv_heads = rng.choice([1, 2, 4, 8])
        ctx = _log_int(rng, 1, 4096 if dtype == "fp32" else 32768)
        nodes = _log_int(rng, 1, 32 if dtype == "fp32" else 96)
        # at most half the tokens, and a quarter of the score products, of the largest listed case
        batch = _log_int(rng, 1, max(1, min(128, (8 * 16384 if dtype == "fp32" else 8 * 196608) // (ctx * kv_heads))))
        group = rng.choice([1, 2, 3, 4, 8])
        while batch * ctx * kv_heads * group * nodes > (1 << 26 if dtype == "fp32" else 1 << 28):
            nodes = max(1, nodes // 2)
            if nodes == 1:
                break
        return {"op": op, "dtype": dtype, "cache": cache, "heads": kv_heads * group, "kv_heads": kv_heads,
                "head_dim": rng.choice([64, 128, 128]), "batch": batch, "block_size": rng.choice([16, 32, 64, 256]),
                "ctx_min": rng.choice([ctx, max(1, ctx // 7)]), "ctx_max": ctx, "nodes_min": rng.choice([1, nodes]),
                "nodes_max": nodes, "lens_seed": seed}
    if op in ("metadata", "accept"):
        nodes = _log_int(rng, 1, 96)
        c = {"op": op, "batch": _log_int(rng, 1, 256), "block_size": rng.choice([16, 32, 64, 256]), "ctx_min": 1,
             "ctx_max": _log_int(rng, 1, 8192), "nodes_min": rng.choice([1, nodes]), "nodes_max": nodes,
             "lens_seed": seed}
        return dict(c, max_path=rng.randint(1, 9)) if op == "accept" else c
    c = {"op": op, "layers": rng.choice([28, 36]), "kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 128]),
         "dtype": rng.choice(["bf16", "fp16", "fp32"]), "block_size": rng.choice([16, 32])}
    row = c["layers"] * c["kv_heads"] * c["head_dim"] * DTYPES[c["dtype"]].itemsize  # bytes of a token's keys
    if op == "copy":
        pairs = _log_int(rng, 1, max(1, min(512, 210_000_000 // (row * c["block_size"]))))
        return dict(c, pages=3 * pairs + rng.randint(1, 40), pairs=pairs)
    return dict(c, batch=_log_int(rng, 1, max(1, min(253, 210_000_000 // (row * 8)))), nodes=rng.randint(10, 33),
                max_path=rng.randint(2, 9), lens_seed=seed)


def _lengths(case):
    """(cached tokens before the tree, nodes of the tree) of each sequence."""
    r = random.Random(case["lens_seed"])
    return ([r.randint(case["ctx_min"], case["ctx_max"]) for _ in range(case["batch"])],
            [r.randint(case["nodes_min"], case["nodes_max"]) for _ in range(case["batch"])])


def _path_lengths(case):
    """Accepted nodes of each sequence of a move: the root, which stays, and up to max_path - 1 others."""
    r = random.Random(case["lens_seed"])
    return [r.randint(1, case["max_path"]) for _ in range(case["batch"])]


# ------------------------------------------------------------------------------ inputs
def _trees(r, nodes):
    """The parent of each node within its tree (-1 for the root), parents before children, at most 8 levels."""
    trees = []
    for n in nodes:
        parent, depth = [-1], [0]
        for j in range(1, n):
            p = r.randrange(j)
            while depth[p] >= 7:
                p = parent[p]
            parent.append(p)
            depth.append(depth[p] + 1)
        trees.append(parent)
    return trees


def _words(trees, width):
    """Ancestor masks (a node sees itself and its ancestors), `width` words of 64 nodes in two's complement."""
    rows = []
    for parent in trees:
        bits = []
        for j, p in enumerate(parent):
            bits.append((bits[p] if p >= 0 else 0) | (1 << j))
            ws = [(bits[j] >> (64 * w)) & ((1 << 64) - 1) for w in range(width)]
            rows.append([w - (1 << 64) if w >> 63 else w for w in ws])
    return rows


def _starts(nodes):
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    return cu


def _tables(lens, block_size, gen, spare=3):
    """Block tables over a random permutation of the physical pages, padded with -1; (tables, pages)."""
    blocks = [-(-n // block_size) for n in lens]
    pages = sum(blocks) + spare
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    count = torch.tensor(blocks, device="cuda")
    at = torch.arange(max(blocks), device="cuda")[None, :]
    idx = (count.cumsum(0) - count)[:, None] + at
    return torch.where(at < count[:, None], perm[idx.clamp(max=pages - 1)], -1).contiguous(), pages


def _quantise(x, cache):
    """(values, scales) of a cache x (pages, rows, heads, head_dim), as the append writes them."""
    if cache == "fp8_per_tensor":
        s = (x.abs().amax() / 448.0).float().reshape(1)
        return (x.float() / s).clamp(-448, 448).to(torch.float8_e4m3fn), s
    s = torch.empty(x.shape[:3], dtype=torch.float32, device=x.device)
    v = torch.empty(x.shape, dtype=torch.int8 if cache.startswith("int8") else torch.float8_e4m3fn, device=x.device)
    for i in range(0, x.shape[0], 512):  # in parts: the 32-bit copy of a whole cache is large
        y = x[i:i + 512].float()
        a = y.abs().amax(-1)
        if cache.startswith("int8"):
            s[i:i + 512] = (a / 127.0).clamp(min=1e-6)
            v[i:i + 512] = (y / s[i:i + 512, ..., None]).round().clamp(-128, 127).to(torch.int8)
        else:
            s[i:i + 512] = a / 448.0
            v[i:i + 512] = (y / s[i:i + 512, ..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return v, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    s = dict(case)
    cuda = lambda v, t: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    if case["op"] in ("copy", "move"):
        if case["op"] == "copy":
            pages, bs = case["pages"], case["block_size"]
            perm = torch.randperm(pages, generator=gen, device="cuda")
            # sources may repeat (a fork's children), destinations are free pages
            s["src"] = perm[:case["pairs"]].contiguous() if case["pairs"] > 8 else perm[:1].repeat(case["pairs"])
            s["dst"] = perm[pages - case["pairs"]:].contiguous()
        else:
            # page 0 is nobody's; a tree's nodes lie on pages of their own, the accepted branch behind the
            # rows it moves to, so that a second pass finds what the first one found
            bs, nodes = case["block_size"], case["nodes"]
            per = -(-(nodes + bs) // bs)
            pages = 1 + case["batch"] * per
            perm = (1 + torch.randperm(pages - 1, generator=gen, device="cuda")).tolist()
            src, dst = [], []
            for b, n in enumerate(_path_lengths(case)):
                first, mine = r.randrange(bs), perm[b * per:(b + 1) * per]
                slot = lambda j: mine[(first + j) // bs] * bs + (first + j) % bs  # noqa: E731,B023
                path = sorted(r.sample(range(case["max_path"], nodes), min(n, nodes - case["max_path"]) - 1))
                pad = [-1] * (case["max_path"] - 1 - len(path))
                src.append([slot(j) for j in path] + pad)
                dst.append([slot(1 + k) for k in range(len(path))] + pad)
            s["src"], s["dst"] = cuda(src, torch.int64), cuda(dst, torch.int64)
        s["kv"] = torch.randn(2, case["layers"], pages, bs, case["kv_heads"], case["head_dim"], generator=gen,
                              device="cuda", dtype=DTYPES[case["dtype"]])
        return s
    prefix, nodes = _lengths(case)
    trees, cu = _trees(r, nodes), _starts(nodes)
    width = -(-max(nodes) // 64)
    s["tables"], pages = _tables([a + b for a, b in zip(prefix, nodes)], case["block_size"], gen)
    s["cu"] = cuda(cu, torch.int32)
    s["prefix"] = cuda(prefix, torch.int64)
    s["parents"] = cuda([p for t in trees for p in t], torch.int32)
    # the plan of a padded batch: the sequence and the node of each row
    s["row_seq"] = cuda([b for b, n in enumerate(nodes) for _ in range(n)], torch.int64)
    s["row_node"] = cuda([j for n in nodes for j in range(n)], torch.int64)
    s["most"] = max(nodes)
    if case["op"] == "accept":
        # drafted tokens, and the target model's: along one branch they agree with the drafts mostly
        draft = [r.randrange(VOCAB) for _ in range(cu[-1])]
        target = [r.randrange(VOCAB) for _ in range(cu[-1])]
        for b, t in enumerate(trees):
            j = len(t) - 1
            while j > 0:
                if r.random() < 0.85:
                    target[cu[b] + t[j]] = draft[cu[b] + j]
                j = t[j]
        s["draft"], s["target"] = cuda(draft, torch.int64), cuda(target, torch.int64)
    if case["op"] == "attention":
        t = DTYPES[case["dtype"]]
        s["mask"] = cuda(_words(trees, width), torch.int64)
        s["lens"] = cuda([a + b for a, b in zip(prefix, nodes)], torch.int64)
        s["trees"] = trees  # host copy, as the drafting program has it
        s["scale"] = case["head_dim"] ** -0.5
        s["query"] = torch.randn(cu[-1], case["heads"], case["head_dim"], generator=gen, device="cuda", dtype=t)
        # heads of different sharpness: some attend broadly, some to a few tokens
        s["query"] *= torch.linspace(0.5, 3.0, case["heads"], device="cuda", dtype=t)[None, :, None]
        for name in ("k", "v"):
            x = torch.randn(pages, case["block_size"], case["kv_heads"], case["head_dim"], generator=gen,
                            device="cuda", dtype=torch.bfloat16 if case["cache"] != "auto" else t)
            x, sc = (x, None) if case["cache"] == "auto" else _quantise(x, case["cache"])
            s[name], s[name + "_scale"] = x, sc
    return s


# ------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        attention, kv_cache = _framework()
        if s["op"] == "attention":
            return attention.paged_attention_tree(
                s["query"], s["k"], s["v"], s["tables"], s["lens"], s["cu"], s["mask"], s["scale"], s["heads"],
                s["kv_heads"], s["head_dim"], s["block_size"], s["k_scale"], s["v_scale"], s["cache"])
        if s["op"] == "metadata":
            m = kv_cache.tree_metadata(s["parents"], s["cu"], s["prefix"], s["tables"], s["block_size"], s["most"])
            return {"slots": m.slot_mapping, "lens": m.context_lens, "positions": m.positions, "mask": m.tree_mask}
        if s["op"] == "accept":
            a = kv_cache.tree_accept(s["draft"], s["target"], s["parents"], s["cu"], s["prefix"], s["tables"],
                                     s["block_size"], s["max_path"])
            return {"count": a.num_accepted, "nodes": a.accepted_nodes, "tokens": a.tokens, "lens": a.context_lens,
                    "src": a.src_slots, "dst": a.dst_slots}
        cache = kv_cache.KVCache(s["kv"], None, None, "auto", s["block_size"])
        if s["op"] == "copy":
            kv_cache.copy_kv_pages(cache, s["src"], s["dst"])
        else:
            kv_cache.move_kv_rows(cache, s["src"], s["dst"])
        return s["kv"]
    if s["op"] == "attention":
        return _plain_attention(s)
    if s["op"] == "metadata":
        return _plain_metadata(s)
    if s["op"] == "accept":
        return _plain_accept(s)
    kv = s["kv"]
    if s["op"] == "copy":
        kv[:, :, s["dst"]] = kv[:, :, s["src"]]
    else:  # an entry of -1 is no move: nobody's row 0 is copied onto itself
        rows = kv.view(kv.shape[0], kv.shape[1], -1, *kv.shape[4:])
        rows[:, :, s["dst"].reshape(-1).clamp(min=0)] = rows[:, :, s["src"].reshape(-1).clamp(min=0)]
    return kv


def _plain_attention(s):
    """Padded batch: gathered pages in 32 bits, masked scores, softmax, product with the values."""
    tables, lens, cu, most = s["tables"].long().clamp(min=0), s["lens"], s["cu"].long(), s["most"]
    batch, h, g, d = s["batch"], s["kv_heads"], s["heads"] // s["kv_heads"], s["head_dim"]

    def gather(x, sc):
        x = x[tables].float()  # (batch, blocks, rows, heads, head_dim)
        if sc is not None:
            x = x * (sc if sc.numel() == 1 else sc[tables][..., None])
        return x.reshape(batch, -1, h, d).transpose(1, 2)

    at = torch.arange(tables.shape[1] * s["block_size"], device="cuda")
    nodes = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + torch.arange(most, device="cuda")).clamp(max=s["query"].shape[0] - 1)  # (batch, most)
    j = at[None, :] - (lens - nodes)[:, None]  # the node at each cached position, below 0 in the prefix
    words = s["mask"][row].gather(2, (j.clamp(min=0) >> 6).clamp(max=s["mask"].shape[1] - 1)[:, None, :].expand(-1, most, -1))
    seen = ((words >> (j.clamp(min=0) & 63)[:, None, :]) & 1).bool() | (j < 0)[:, None, :]
    seen = (seen & (j < nodes[:, None])[:, None, :])[:, None, :, None, :]  # (batch, 1, most, 1, tokens)
    q = s["query"][row].float().reshape(batch, most, h, g, d).transpose(1, 2).reshape(batch, h, most * g, d)
    p = (q @ gather(s["k"], s["k_scale"]).transpose(2, 3)) * s["scale"]
    p = p.view(batch, h, most, g, -1).masked_fill_(~seen, float("-inf")).view(batch, h, most * g, -1)
    p = (p - p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    # positions behind a sequence's end hold other sequences' rows or none: they count as zeros
    v = gather(s["v"], s["v_scale"]).masked_fill((at[None, :] >= lens[:, None])[:, None, :, None], 0.0)
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = o.view(batch, h, most, g, d).transpose(1, 2).reshape(batch, most, h * g, d)
    return o[s["row_seq"], s["row_node"]].to(s["query"].dtype)


def _padded(s, x, fill):
    """Values of the rows as (batch, most)."""
    y = torch.full((s["batch"], s["most"]), fill, dtype=torch.int64, device="cuda")
    y[s["row_seq"], s["row_node"]] = x.long()
    return y


def _slot(s, seq, pos):
    return s["tables"][seq, pos // s["block_size"]].long() * s["block_size"] + pos % s["block_size"]


def _plain_metadata(s):
    n = s["most"]
    parent = _padded(s, s["parents"], -1)
    at = torch.arange(n, device="cuda")
    sees = ((parent[:, :, None] == at) | (at[:, None] == at)).float()  # itself and its parent
    for _ in range((n - 1).bit_length()):  # the transitive closure, by squaring
        sees = (sees @ sees > 0).float()
    sees = sees[s["row_seq"], s["row_node"]].long()  # (rows, n)
    positions = s["prefix"][s["row_seq"]] + sees.sum(-1) - 1
    width = -(-n // 64)
    bits = torch.nn.functional.pad(sees, (0, 64 * width - n)).view(-1, width, 64) << torch.arange(64, device="cuda")
    where = s["prefix"][s["row_seq"]] + s["row_node"]
    nodes = s["cu"][1:] - s["cu"][:-1]
    return {"slots": _slot(s, s["row_seq"], where), "lens": s["prefix"] + nodes, "positions": positions,
            "mask": bits.sum(-1)}


def _plain_accept(s):
    batch, n, most = s["batch"], s["most"], s["max_path"]
    parent, draft, target = _padded(s, s["parents"], -2), _padded(s, s["draft"], -1), _padded(s, s["target"], -1)
    at = torch.arange(n, device="cuda")
    cur = torch.zeros(batch, 1, dtype=torch.int64, device="cuda")  # the root is taken
    path, on = [cur], torch.ones_like(cur, dtype=torch.bool)
    for _ in range(most - 1):  # a level a step: what is taken next hangs on what was taken
        fits = (parent == cur) & (draft == target.gather(1, cur)) & (at > 0) & on
        nxt = torch.where(fits, at, n).amin(1, keepdim=True)  # the lowest index among equals
        on = nxt < n
        cur = torch.where(on, nxt, cur)
        path.append(torch.where(on, nxt, -1))
    path = torch.cat(path, 1)
    taken = path >= 0
    count = taken.sum(1)
    seq = torch.arange(batch, device="cuda")[:, None]
    k = torch.arange(most, device="cuda")
    moved = taken & (path != k)
    last = s["prefix"][:, None] + (s["cu"][1:] - s["cu"][:-1]).long()[:, None] - 1
    src = _slot(s, seq, (s["prefix"][:, None] + path.clamp(min=0)).minimum(last))
    dst = _slot(s, seq, (s["prefix"][:, None] + k).minimum(last))
    return {"count": count.int(), "nodes": path.int(), "tokens": torch.where(taken, target.gather(1, path.clamp(min=0)), -1),
            "lens": s["prefix"] + count, "src": torch.where(moved, src, -1), "dst": torch.where(moved, dst, -1)}


# ------------------------------------------------------------------------------ bytes and operations
def work(case):
    if case["op"] in ("copy", "move"):
        row = 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * DTYPES[case["dtype"]].itemsize
        if case["op"] == "copy":  # a page that several take is read once
            reads = case["pairs"] if case["pairs"] > 8 else 1
            return {"bytes": (reads + case["pairs"]) * row * case["block_size"], "flops": 0}
        rows = sum(min(n, case["nodes"] - case["max_path"]) - 1 for n in _path_lengths(case))
        return {"bytes": 2 * rows * row + 16 * case["batch"] * (case["max_path"] - 1), "flops": 0}
    prefix, nodes = _lengths(case)
    total, batch, width = sum(nodes), case["batch"], -(-max(nodes) // 64)
    if case["op"] == "metadata":  # parents, starts, lengths, the trees' pages; slots, positions, masks, lengths
        return {"bytes": total * (4 + 8 + 8 + 8 * width) + batch * (4 + 8 + 8) + 4 * total // case["block_size"], "flops": 0}
    if case["op"] == "accept":  # tokens and parents; the paths and their moves
        return {"bytes": total * (8 + 8 + 4) + batch * (4 + 8) + batch * (4 + 8) + batch * case["max_path"] * (4 + 8 + 8 + 8),
                "flops": 0}
    t = DTYPES[case["dtype"]].itemsize
    row = case["kv_heads"] * (case["head_dim"] * (t if case["cache"] == "auto" else 1) + (4 if "token" in case["cache"] else 0))
    tokens = sum(prefix) + total
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(prefix, nodes))
    return {"bytes": 2 * tokens * row + 2 * total * case["heads"] * case["head_dim"] * t + total * 8 * width
            + 4 * (tokens // case["block_size"] + batch), "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """Each sequence for itself, from the operators' definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "copy":
        kv = s["kv"].clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            kv[:, :, b].copy_(s["kv"][:, :, a])
        return kv.to(torch.float64)
    if case["op"] == "move":
        bs, kv = case["block_size"], s["kv"].clone()
        for a, b in zip(s["src"].reshape(-1).tolist(), s["dst"].reshape(-1).tolist()):
            if a >= 0:
                kv[:, :, b // bs, b % bs].copy_(s["kv"][:, :, a // bs, a % bs])
        return kv.to(torch.float64)
    return None  # whole numbers


def _exact_attention(s):
    bs, g, first, out = s["block_size"], s["heads"] // s["kv_heads"], 0, []
    for b, parent in enumerate(s["trees"]):
        n, length = len(parent), int(s["lens"][b])
        t = torch.arange(length, device="cuda")
        page, at = s["tables"][b].long()[t // bs], t % bs
        hidden = torch.zeros(n, length, dtype=torch.bool, device="cuda")
        for i in range(n):
            sees, j = set(), i
            while j >= 0:
                sees.add(j)
                j = parent[j]
            for j in range(n):
                if j not in sees:
                    hidden[i, length - n + j] = True
        rows = []
        for h in range(s["kv_heads"]):
            k, v = (s[c][page, at, h].double() for c in "kv")
            if s["k_scale"] is not None:
                ks, vs = (s[c + "_scale"] if s[c + "_scale"].numel() == 1 else s[c + "_scale"][page, at, h, None] for c in "kv")
                k, v = k * ks.double(), v * vs.double()
            q = s["query"][first:first + n, h * g:(h + 1) * g].double()
            x = torch.einsum("ngd,td->ngt", q, k) * s["scale"]
            x = torch.softmax(x.masked_fill(hidden[:, None, :], -math.inf), -1)
            rows.append(torch.einsum("ngt,td->ngd", x, v))
        out.append(torch.cat(rows, 1))
        first += n
    return torch.cat(out, 0)
