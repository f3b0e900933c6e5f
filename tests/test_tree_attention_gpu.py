"""paged_attention_tree against the 64-bit oracle: types, cache modes, head layouts, page
sizes, lengths from nothing to long, masks that leave rows empty, and whatever a row does
not see holding infinities and NaN."""
import math
import random

import pytest
import torch

from conftest import mkv_module
from oracle.tree_oracle import mask_words, paged_tree_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def trees(r, nodes, depth=8):
    out = []
    for n in nodes:
        sees = []
        for j in range(n):
            sees.append({j} | (sees[r.randrange(j)] if j else set()))
            while len(sees[j]) > depth:
                sees[j] = {j} | sees[min(sees[j])]
        out.append(sees)
    return out


def quantise(x, mode):
    y = x.float()
    if mode == "fp8_per_tensor":
        s = (y.abs().amax() / 448).reshape(1)
        return (y / s).to(torch.float8_e4m3fn), s
    s = y.abs().amax(-1).clamp(min=1e-6) / (127 if mode.startswith("int8") else 448)
    y = y / s[..., None]
    return (y.round().clamp(-128, 127).to(torch.int8) if mode.startswith("int8") else y.to(torch.float8_e4m3fn)), s


class Case:
    """A batch over a random permutation of pages; what no row sees is NaN or infinite."""

    def __init__(self, seed, prefix, nodes, H, KVH, D, BS, dtype, mode="auto", visible=None, index=torch.int64,
                 spread=1.0, poison=True, missing=(), words=None, offset=0.0):
        r = random.Random(seed)
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.H, self.KVH, self.D, self.BS, self.mode, self.dtype = H, KVH, D, BS, mode, dtype
        self.B = len(prefix)
        lens = [a + b for a, b in zip(prefix, nodes)]
        blocks = [-(-n // BS) for n in lens]
        NB = sum(blocks) + 3
        perm = torch.randperm(NB, generator=g, device=DEV).tolist()
        width = max(max(blocks), 1) + 1
        bt = torch.full((self.B, width), -1)
        at = 0
        for b, k in enumerate(blocks):
            bt[b, :k] = torch.tensor(perm[at:at + k])
            at += k
        for b, k in missing:
            bt[b, k] = -1 if (b + k) % 2 else NB + 5
        self.cu = [0]
        for n in nodes:
            self.cu.append(self.cu[-1] + n)
        total = self.cu[-1]
        self.visible = visible if visible is not None else trees(r, nodes)
        self.words = words or max(1, -(-max(nodes) // 64))
        self.q = (torch.randn(total, H, D, generator=g, device=DEV) * spread).to(dtype)
        shape = (NB, BS, KVH, D)
        k = torch.randn(shape, generator=g, device=DEV) + offset
        v = torch.randn(shape, generator=g, device=DEV) + offset
        self.ks = self.vs = None
        if mode == "auto":
            self.k, self.v = k.to(dtype), v.to(dtype)
        else:
            self.k, self.ks = quantise(k.to(BF16), mode)
            self.v, self.vs = quantise(v.to(BF16), mode)
        self.bt = bt.to(DEV, torch.int32 if index == torch.int64 else torch.int64)
        self.lens = torch.tensor(lens, dtype=index, device=DEV)
        self.cut = torch.tensor(self.cu, dtype=torch.int32 if index == torch.int64 else torch.int64, device=DEV)
        self.mask = mask_words(self.visible, self.words).to(DEV).reshape(total, self.words)
        self.scale = 1.0 / math.sqrt(D)
        if poison:
            self.poison(bt, lens, NB)

    def poison(self, bt, lens, NB):
        """NaN (or infinity) in every cached row that no sequence holds."""
        used = torch.zeros(NB, self.BS, dtype=torch.bool)
        for b, n in enumerate(lens):
            for t in range(n):
                page = int(bt[b, t // self.BS])
                if 0 <= page < NB:
                    used[page, t % self.BS] = True
        dead = (~used).to(DEV)
        if self.mode == "int8_per_token_head":
            self.ks[dead], self.vs[dead] = float("nan"), float("inf")
            return
        if self.mode != "auto":
            for c in (self.k, self.v):
                c.view(torch.uint8)[dead] = 0x7F  # the NaN of e4m3
            if self.mode != "fp8_per_tensor":
                self.ks[dead], self.vs[dead] = float("inf"), float("nan")
            return
        self.k[dead], self.v[dead] = float("nan"), float("inf")

    def run(self, attn, q=None, out=None):
        return attn.paged_attention_tree(self.q if q is None else q, self.k, self.v, self.bt, self.lens, self.cut,
                                         self.mask, self.scale, self.H, self.KVH, self.D, self.BS, self.ks, self.vs,
                                         self.mode, out=out)

    def ref(self):
        return paged_tree_ref(self.q, self.k, self.v, self.bt, self.lens, self.cu, self.visible, self.scale,
                              self.ks, self.vs)

    def check(self, got):
        """|error| <= u |o| (rounding the output) + A (u_p + 2 e + T 2^-24 + 2^-20), A = sum_t
        w_t |v_t|: u_p rounds the weights to 16 bits before the product with the values; e is
        the error of a score, at most (D + 4) 2^-24 sum_d |q_d k_d| scale for the sum and
        its scaling; T 2^-24 for summing T terms; 2^-20 for the exponential (2^-22 each in
        p and in its sum, and in the joining of parts). An f16 output below 2^-14 is a
        multiple of 2^-24 (a subnormal), so its rounding is off by up to 2^-25 whatever its
        size: a column in which the one token that weighs holds an int8 0 is such a case."""
        ref, mag, mags = self.ref()
        u = torch.finfo(self.dtype).eps / 2
        T = int(max(self.lens.max(), 1))
        e = (self.D + 4) * 2.0 ** -24 * mags[..., None]
        tol = u * ref.abs() + mag * ((u if self.dtype != F32 else 0.0) + 2 * e + T * 2.0 ** -24 + 2.0 ** -20)
        tol = tol + (2.0 ** -25 if self.dtype == F16 else 1e-38)
        assert got.shape == self.q.shape and got.dtype == self.dtype
        err = (got.double() - ref).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num(1e9).max()):.3g} "
                               f"times the bound, first at {bad.nonzero()[0].tolist()}")


MODES = [(BF16, "auto"), (F16, "auto"), (F32, "auto"), (BF16, "fp8_per_tensor"), (F16, "fp8_per_token_head"),
         (BF16, "int8_per_token_head"), (F32, "fp8_per_token_head"), (F16, "int8_per_token_head"),
         (F32, "int8_per_token_head"), (BF16, "fp8_per_token_head"), (F16, "fp8_per_tensor")]


@pytest.mark.parametrize("dtype,mode", MODES)
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 128), (4, 4, 64), (6, 2, 128), (16, 1, 64)])
def test_types_and_heads(attn, dtype, mode, H, KVH, D):
    c = Case(1, [77, 0, 300, 15], [9, 1, 16, 5], H, KVH, D, 16, dtype, mode)
    c.check(c.run(attn))


@pytest.mark.parametrize("mode", ["auto", "fp8_per_tensor", "int8_per_token_head"])
@pytest.mark.parametrize("prefix,nodes", [
    ([0], [1]), ([1], [1]), ([15], [1]), ([16], [2]), ([63], [1]), ([64], [1]), ([127], [3]), ([128], [64]),
    ([0, 0, 0], [0, 1, 0]), ([5, 1000, 0, 130], [3, 1, 64, 33]), ([1100], [65]), ([61], [130]), ([0], [97]),
    ([2000] * 3 + [1] * 9, [1] * 12)])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(attn, mode, prefix, nodes, D):
    c = Case(2, prefix, nodes, 8, 2, D, 16, BF16, mode)
    c.check(c.run(attn))


@pytest.mark.parametrize("BS", [1, 7, 8, 16, 48, 64, 128, 256])
@pytest.mark.parametrize("dtype,mode", [(BF16, "auto"), (F16, "fp8_per_token_head"), (BF16, "int8_per_token_head")])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(attn, BS, dtype, mode, D):
    c = Case(3, [300, 7, 129], [20, 3, 40], 8, 2, D, BS, dtype, mode)
    c.check(c.run(attn))


@pytest.mark.parametrize("D", [16, 48, 80, 96, 256])
@pytest.mark.parametrize("dtype,mode", [(BF16, "auto"), (F32, "auto"), (F16, "int8_per_token_head")])
def test_other_head_dims(attn, D, dtype, mode):
    c = Case(4, [150, 33], [11, 6], 6, 2, D, 16, dtype, mode)
    c.check(c.run(attn))


@pytest.mark.parametrize("H,KVH", [(7, 1), (10, 2), (32, 1), (160, 1), (3, 3)])
def test_groups(attn, H, KVH):
    """Also groups that do not divide the row tile, and rows beyond one tile."""
    c = Case(5, [210, 40], [13, 30], H, KVH, 128, 16, BF16)
    c.check(c.run(attn))


@pytest.mark.parametrize("dtype,mode", [(BF16, "auto"), (BF16, "fp8_per_tensor"), (F32, "auto")])
def test_any_mask(attn, dtype, mode):
    """Masks that are no trees: rows that see nothing of the tree, later nodes, one node only,
    all; over a prefix and without one (then a row may see nothing at all: zeros)."""
    r = random.Random(6)
    nodes, prefix = [20, 70, 3, 40], [0, 100, 0, 0]
    visible = [[set(j for j in range(n) if r.random() < p) for p in [r.choice([0, 0.1, 0.5, 1]) for _ in range(n)]]
               for n in nodes]
    visible[2] = [set(), {2}, set()]
    c = Case(6, prefix, nodes, 8, 2, 128, 16, dtype, mode, visible=visible)
    got = c.run(attn)
    c.check(got)
    assert (got[c.cu[2]] == 0).all() and (got[c.cu[2] + 2] == 0).all()


@pytest.mark.parametrize("dtype,mode", [(BF16, "auto"), (F16, "auto"), (F32, "auto"), (BF16, "fp8_per_tensor"),
                                        (BF16, "fp8_per_token_head"), (F16, "int8_per_token_head")])
@pytest.mark.parametrize("prefix", [0, 40, 120, 700])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_nodes_may_hold_anything(attn, dtype, mode, prefix, D):
    """A drafted branch that overflowed reaches only the rows that see it."""
    n, sick = 12, 5
    visible = [[{0, j} for j in range(n)]]
    for j in range(n):
        if j != sick:
            visible[0][j].discard(sick)
    c = Case(7, [prefix], [n], 8, 2, D, 16, dtype, mode, visible=visible)
    t = prefix + sick
    page, at = int(c.bt[0, t // 16]), t % 16
    if mode == "int8_per_token_head":
        c.ks[page, at], c.vs[page, at] = float("nan"), float("inf")
    elif mode != "auto":
        c.k.view(torch.uint8)[page, at] = 0x7F
        c.v.view(torch.uint8)[page, at, :, ::3] = 0xFF
    else:
        c.k[page, at] = float("nan")
        c.v[page, at, :, ::2], c.v[page, at, :, 1::2] = float("inf"), float("nan")
    got = c.run(attn)
    rows = [j for j in range(n) if j != sick]
    assert torch.isfinite(got[rows]).all()
    assert torch.isnan(got[sick]).any()
    c.visible[0][sick] = {0}  # the rest of the check leaves that row out
    ref, _, _ = c.ref()
    got = got.clone()
    got[sick] = ref[sick].to(dtype)
    c.check(got)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("prefix", [3, 400])
def test_infinite_values_that_are_seen(attn, dtype, prefix):
    """An infinite value of a node that rows see makes their outputs infinite in that column
    alone (its weight is positive)."""
    c = Case(8, [prefix], [6], 4, 2, 128, 16, dtype, visible=[[set(range(j + 1)) for j in range(6)]])
    t = prefix + 3
    c.v[int(c.bt[0, t // 16]), t % 16, 1, 17] = -float("inf")
    got = c.run(attn)
    inf = torch.zeros_like(got, dtype=torch.bool)
    inf[3:, 2:, 17] = True
    assert (got[inf] == -float("inf")).all() and torch.isfinite(got[~inf]).all()


def test_scores_of_minus_infinity(attn):
    """A visible score of -inf weighs nothing next to finite ones; where all are, 0 / 0."""
    c = Case(9, [2], [3], 2, 1, 64, 16, F32, visible=[[{0}, {0, 1}, {2}]])
    c.q.abs_()
    for t in (0, 1, 2, 4):
        c.k[int(c.bt[0, 0]), t] = -float("inf")
    got = c.run(attn)
    assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all()
    v = c.v[int(c.bt[0, 0]), 3, 0]
    assert torch.allclose(got[1], v.expand(2, -1), rtol=2 ** -20, atol=0)


@pytest.mark.parametrize("dtype,mode", [(BF16, "auto"), (F16, "fp8_per_tensor")])
@pytest.mark.parametrize("BS", [16, 64, 48])
def test_missing_pages(attn, dtype, mode, BS):
    c = Case(10, [700, 90], [17, 5], 8, 2, 128, BS, dtype, mode, missing=[(0, 0), (0, 3), (1, 1)], poison=False)
    c.check(c.run(attn))


def test_table_narrower_than_the_context(attn):
    c = Case(11, [300], [9], 8, 2, 128, 16, BF16, poison=False)
    c.bt = c.bt[:, :12].contiguous()
    c.check(c.run(attn))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_strides_index_types_and_out(attn, index):
    """Queries and outputs as slices of wider tensors, a mask that is a slice of a wider one,
    a table with spare columns, either index type."""
    c = Case(12, [140, 33, 900], [10, 70, 1], 8, 2, 128, 16, BF16, index=index)
    total = c.cu[-1]
    fused = torch.randn(total + 3, 12, 128, device=DEV).to(BF16)
    fused[:total, 2:10] = c.q
    wide = torch.zeros(total, 5, dtype=torch.int64, device=DEV)
    wide[:, :c.words] = c.mask
    c.mask = wide[:, :c.words]
    out = torch.full((total, 9, 130), 7.0, device=DEV, dtype=BF16)
    got = c.run(attn, q=fused[:total, 2:10], out=out[:, 1:, :128])
    assert got.data_ptr() == out[:, 1:].data_ptr()
    c.check(got)
    assert (out[:, 0] == 7).all() and (out[:, :, 128:] == 7).all()
    odd = torch.randn(total, 8, 131, device=DEV).to(BF16)  # rows that no vector load fits
    odd[..., 1:129] = c.q
    c.check(c.run(attn, q=odd[..., 1:129]))
    turned = c.q.transpose(1, 2).contiguous().transpose(1, 2)  # head_dim not innermost
    c.check(c.run(attn, q=turned))


def test_rows_of_no_sequence_are_left(attn):
    """A padded batch: rows behind the last sequence keep what `out` held."""
    c = Case(13, [50, 200], [4, 6], 8, 2, 128, 16, BF16)
    q = torch.cat([c.q, torch.full((5, 8, 128), float("nan"), device=DEV, dtype=BF16)])
    out = torch.full_like(q, 3.0)
    c.mask = torch.cat([c.mask, torch.full((5, c.words), -1, device=DEV, dtype=torch.int64)])
    c.run(attn, q=q, out=out)
    c.check(out[:10])
    assert (out[10:] == 3).all()


@pytest.mark.parametrize("dtype,mode", [(BF16, "auto"), (BF16, "fp8_per_tensor"), (F16, "int8_per_token_head")])
@pytest.mark.parametrize("nodes", [1, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_sharp_and_flat_scores(attn, dtype, mode, nodes, D):
    """Queries 30 times as large (weights down to nothing), and all keys equal (all weights
    equal, values with a common offset)."""
    c = Case(14, [1500, 3], [nodes, nodes], 8, 2, D, 64, dtype, mode, spread=30.0)
    c.check(c.run(attn))
    c = Case(15, [1500, 3], [nodes, nodes], 8, 2, D, 64, dtype, mode, spread=0.0, offset=2.0)
    c.check(c.run(attn))


def test_long_context(attn):
    """One token and a tree over 33 thousand tokens (many parts of one unit)."""
    for nodes in ([1], [24]):
        c = Case(16, [33001], nodes, 4, 1, 128, 256, BF16)
        c.check(c.run(attn))


def test_many_sequences(attn):
    """More sequences than a CTA has threads, most of them short, some without nodes."""
    r = random.Random(17)
    B = 333
    c = Case(17, [r.choice([0, 1, 17, 40]) for _ in range(B)], [r.choice([0, 1, 2, 5]) for _ in range(B)], 4, 2, 64,
             16, BF16)
    c.check(c.run(attn))


@pytest.mark.parametrize("mode", ["auto", "fp8_per_tensor"])
def test_more_sequences_than_any_block_has_threads(attn, mode):
    r = random.Random(26)
    c = Case(26, [r.choice([0, 1, 17, 40]) for _ in range(1100)], [r.choice([0, 1, 2, 5]) for _ in range(1100)], 4, 2, 64,
             16, BF16, mode)
    c.check(c.run(attn))


def test_pages_past_32_bits(attn):
    """A cache of 2^31 + elements: byte and element offsets beyond 32 bits."""
    NB, BS, KVH, D = 70000, 256, 1, 128  # 2.3e9 elements
    k = torch.zeros(NB, BS, KVH, D, dtype=torch.float8_e4m3fn, device=DEV)
    v = torch.zeros(NB, BS, KVH, D, dtype=torch.float8_e4m3fn, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(18)
    pages = [NB - 1, 3, NB - 2]
    for p in pages:
        k[p] = torch.randn(BS, KVH, D, generator=g, device=DEV).to(torch.float8_e4m3fn)
        v[p] = torch.randn(BS, KVH, D, generator=g, device=DEV).to(torch.float8_e4m3fn)
    c = Case(18, [600], [7], 4, 1, 128, 256, BF16, "fp8_per_tensor", poison=False)
    c.k, c.v = k, v
    c.bt = torch.tensor([pages], dtype=torch.int32, device=DEV)
    got = c.run(attn)
    c.k, c.v = k[pages], v[pages]  # the oracle on the three pages alone
    c.bt = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    c.check(got)


def test_negative_and_zero_scales(attn):
    """A score scale below 0 prefers the least alike; 0 makes every weight equal."""
    for dtype, mode in ((BF16, "auto"), (F16, "fp8_per_tensor"), (BF16, "int8_per_token_head"), (F32, "auto")):
        for scale in (-0.09, 0.0):
            c = Case(22, [200, 3], [9, 20], 8, 2, 128, 16, dtype, mode)
            c.scale = scale
            c.check(c.run(attn))
            if dtype == BF16:  # tiny queries too: their f16 form has a power of two of its own
                c.q = (c.q.float() * 2.0 ** -70).to(BF16)
                c.check(c.run(attn))


@pytest.mark.parametrize("size", [1e-6, 1e4])
@pytest.mark.parametrize("mode", ["fp8_per_tensor", "int8_per_token_head", "fp8_per_token_head"])
def test_sizes_of_queries_and_values(attn, size, mode):
    """Queries and value scales far from 1 (f16 operands hold only so much)."""
    c = Case(23, [300, 40], [12, 3], 8, 2, 128, 16, BF16, mode)
    c.q = (c.q.float() * size).to(BF16)
    c.ks = c.ks / size
    c.vs = c.vs * size
    c.check(c.run(attn))


def test_value_scales_of_every_size(attn):
    """Per-(token, head) value scales that differ by 2^20 within and between tiles, up and down."""
    c = Case(24, [1000], [30], 8, 2, 128, 16, BF16, "int8_per_token_head")
    g = torch.Generator(device=DEV).manual_seed(24)
    c.vs = c.vs * torch.exp2(torch.randint(-10, 11, c.vs.shape, generator=g, device=DEV).float())
    at = c.bt[0].long()
    c.vs[at[:20]] *= 2.0 ** 12
    c.vs[at[40:50]] *= 2.0 ** -12
    c.check(c.run(attn))


@pytest.mark.parametrize("dtype,mode,nodes", [(BF16, "auto", 3), (BF16, "auto", 40), (BF16, "fp8_per_tensor", 8),
                                              (F32, "auto", 4)])
def test_deterministic_streams_and_graphs(attn, dtype, mode, nodes):
    """The same bits from call to call, from two streams at once, and from two graphs that
    are captured one after the other and replayed side by side."""
    c = Case(19, [5000, 700, 12], [nodes, 1, nodes], 8, 2, 128, 16, dtype, mode)
    want = c.run(attn)
    c.check(want)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(c.run(attn))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs, held = [], []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            held.append(c.run(attn))
        graphs.append(g)
    for o in held:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in held)


def test_single_tokens_agree_with_decode(attn):
    """Trees of one node are the decode's single tokens."""
    c = Case(20, [100, 0, 999], [1, 1, 1], 32, 8, 128, 16, BF16, poison=False)
    tree = c.run(attn)
    dec = attn.paged_attention_decode(c.q, c.k, c.v, c.bt, c.lens, c.scale, 32, 8, 128, 16)
    c.check(tree)
    c.check(dec)


def test_attention_module_takes_the_tree_branch(attn):
    c = Case(21, [100, 30], [6, 9], 8, 2, 128, 16, BF16)
    ctx = mkv_module("utils.context")
    layer = attn.Attention(8, 128, 1.0, 2, 16)
    layer.k_cache, layer.v_cache = c.k, c.v
    new_k = torch.randn(15, 2, 128, device=DEV).to(BF16)
    new_v = torch.randn(15, 2, 128, device=DEV).to(BF16)
    kv = mkv_module("engine.kv_cache")
    parents = torch.tensor([-1, 0, 0, 1, 1, 4] + [-1] + list(range(8)), dtype=torch.int32, device=DEV)
    m = kv.tree_metadata(parents, c.cut, c.lens - torch.tensor([6, 9], device=DEV), c.bt, 16, 9)
    try:
        ctx.set_context(True, cu_seqlens_q=c.cut, slot_mapping=m.slot_mapping, context_lens=m.context_lens,
                        block_tables=c.bt, positions=m.positions, tree_mask=m.tree_mask)
        got = layer(c.q, new_k, new_v)
    finally:
        ctx.reset_context()
    assert torch.equal(c.k.view(-1, 2, 128)[m.slot_mapping], new_k)
    c.visible = [[{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 4}, {0, 1, 4, 5}], [set(range(j + 1)) for j in range(9)]]
    c.check(got.view(15, 8, 128))


def test_a_context_without_the_field(attn, monkeypatch):
    """A runner's own context object, made before trees, still decodes."""
    import types
    c = Case(25, [100, 30], [1, 1], 8, 2, 128, 16, BF16, poison=False)
    layer = attn.Attention(8, 128, 1.0, 2, 16)
    layer.k_cache, layer.v_cache = c.k, c.v
    context = types.SimpleNamespace(is_prefill=False, slot_mapping=None, context_lens=c.lens, block_tables=c.bt)
    monkeypatch.setattr(attn, "get_context", lambda: context)
    c.check(layer(c.q, None, None).view(2, 8, 128))


def stale(*shape, dtype):
    """Leaves NaN in the memory that the next tensors of this size are likely to get."""
    held = [torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dtype,mode,D", [(BF16, "auto", 128), (F16, "auto", 64), (F32, "auto", 128),
                                          (BF16, "fp8_per_tensor", 128), (F16, "int8_per_token_head", 64),
                                          (BF16, "auto", 80)])
@pytest.mark.parametrize("front,behind", [(0, 5), (3, 0), (2, 300), (0, 0)])
def test_rows_of_no_sequence_are_zero_without_out(attn, dtype, mode, D, front, behind):
    """A padded batch's rows, before the first and behind the last sequence, are defined: zeros,
    whatever their queries and masks hold, and whatever the memory held."""
    c = Case(27, [50, 0, 2100], [4, 0, 6], 8, 2, D, 16, dtype, mode)
    nan = lambda n: torch.full((n, 8, D), float("nan"), device=DEV, dtype=dtype)  # noqa: E731
    ones = lambda n: torch.full((n, c.words), -1, device=DEV, dtype=torch.int64)  # noqa: E731
    q, mask = torch.cat([nan(front), c.q, nan(behind)]), torch.cat([ones(front), c.mask, ones(behind)])
    cu = c.cut
    c.mask, c.cut = mask, cu + front
    stale(*q.shape, dtype=dtype)
    got = c.run(attn, q=q)
    c.cut = cu
    c.check(got[front:front + 10])
    assert (got[:front] == 0).all() and (got[front + 10:] == 0).all()
    out = torch.full((front + 10 + behind, 9, D + 2), 7.0, dtype=dtype, device=DEV)  # a given `out` keeps its rows
    c.cut = cu + front
    c.run(attn, q=q, out=out[:, 1:, :D])
    c.cut = cu
    c.check(out[front:front + 10, 1:, :D])
    assert (out[:front] == 7).all() and (out[front + 10:] == 7).all()


def test_padding_alone_is_zero(attn):
    """A captured step whose every row is padding (no sequence)."""
    q = torch.full((9, 8, 128), float("nan"), dtype=BF16, device=DEV)
    cache = torch.zeros(3, 16, 2, 128, dtype=BF16, device=DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    stale(9, 8, 128, dtype=BF16)
    got = attn.paged_attention_tree(q, cache, cache, torch.zeros(0, 4, dtype=torch.int32, device=DEV), none,
                                    torch.zeros(1, dtype=torch.int32, device=DEV),
                                    torch.zeros(9, 1, dtype=torch.int64, device=DEV), 0.1, 8, 2, 128, 16)
    assert (got == 0).all()


@pytest.mark.parametrize("captured", [False, True])
def test_a_padded_step_through_two_layers(attn, captured):
    """Attention.forward on a padded tree step: what its padding rows hand to the next layer is
    finite, so that layer's append, which takes its e4m3 scale from all rows of its first step,
    padding included, does not take it from whatever memory held."""
    c = Case(28, [100, 30], [6, 9], 8, 2, 128, 16, BF16, poison=False)
    ctx, kv = mkv_module("utils.context"), mkv_module("engine.kv_cache")
    cache = kv.allocate_kv_cache(2, c.k.shape[0], 16, 2, 128, "fp8_per_tensor", BF16, DEV)
    layers = [attn.Attention(8, 128, 1.0, 2, 16) for _ in range(2)]
    kv.bind_kv_cache(layers, cache)
    pad = 4
    parents = torch.tensor([-1, 0, 0, 1, 1, 4] + [-1] + list(range(8)) + [-1] * pad, dtype=torch.int32, device=DEV)
    q = torch.cat([c.q, torch.ones(pad, 8, 128, dtype=BF16, device=DEV)])
    prefix = c.lens - torch.tensor([6, 9], device=DEV)

    def step():
        m = kv.tree_metadata(parents, c.cut, prefix, c.bt, 16, 9)
        ctx.set_context(True, cu_seqlens_q=c.cut, slot_mapping=m.slot_mapping, context_lens=m.context_lens,
                        block_tables=c.bt, positions=m.positions, tree_mask=m.tree_mask)
        x = layers[0](q, q[:, :2], q[:, 2:4])
        y = layers[1](x.view(-1, 8, 128), x.view(-1, 8, 128)[:, :2], x.view(-1, 8, 128)[:, 2:4])
        return x, y

    try:
        if captured:
            step()
            cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                x, y = step()
            x.fill_(float("nan")), y.fill_(float("nan"))
            graph.replay()
        else:
            stale(19, 8, 128, dtype=BF16)
            x, y = step()
        torch.cuda.synchronize()
    finally:
        ctx.reset_context()
    assert (x[15:] == 0).all() and (y[15:] == 0).all()
    assert torch.isfinite(x).all() and torch.isfinite(y).all()
    assert torch.isfinite(cache.k_scale).all() and torch.isfinite(cache.v_scale).all()


@pytest.mark.parametrize("dtype,mode,D", [(BF16, "auto", 128), (F16, "auto", 64), (BF16, "fp8_per_tensor", 128),
                                          (BF16, "fp8_per_token_head", 64), (F16, "int8_per_token_head", 128)])
@pytest.mark.parametrize("prefix,nodes", [([411], [8]), ([9000, 3, 0, 700], [33, 0, 1, 20]), ([40] * 200, [3] * 200)])
def test_waits_that_run_out_are_seen(attn, dtype, mode, D, prefix, nodes):
    """With a limit of 0 every block gives up before its first wait, with nothing in flight: the
    call ends, all rows of sequences are NaN (split and whole units, over finite values of earlier
    calls in the workspace and the output), other rows are what they are without that, and the
    next call, with the limit as it was, is right."""
    lib = mkv_module("_lib").load()
    c = Case(29, prefix, nodes, 8, 2, D, 16, dtype, mode)
    total = c.cu[-1]
    q = torch.cat([c.q, torch.ones(3, 8, D, dtype=dtype, device=DEV)])
    c.mask = torch.cat([c.mask, torch.zeros(3, c.words, dtype=torch.int64, device=DEV)])
    out = torch.full((total + 3, 8, D), 5.0, dtype=dtype, device=DEV)
    c.run(attn, q=q, out=out)  # leaves finite partial sums where the next call's workspace will be
    c.check(out[:total])
    was = lib.mkv_set_wait_limit(0)
    try:
        given, own = c.run(attn, q=q, out=out.clone()), c.run(attn, q=q)
        torch.cuda.synchronize()
    finally:
        assert lib.mkv_set_wait_limit(was) == 0
    assert torch.isnan(given[:total]).all() and (given[total:] == 5).all()
    assert torch.isnan(own[:total]).all() and (own[total:] == 0).all()
    again = c.run(attn, q=q, out=out)
    c.check(again[:total])


@pytest.mark.parametrize("dtype,mode", [(BF16, "int8_per_token_head"), (F16, "int8_per_token_head"),
                                        (BF16, "fp8_per_token_head"), (F16, "fp8_per_token_head"),
                                        (F32, "int8_per_token_head")])
@pytest.mark.parametrize("prefix", [0, 40, 700])
@pytest.mark.parametrize("log2", [14, 24, 60, 110])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_value_scales_of_any_size(attn, dtype, mode, prefix, log2, D):
    """A node whose (finite) value scale is 2^14 to 2^110 times the others' does not reach the rows
    that do not see it: they are as exact as without it."""
    n, big = 12, 5
    visible = [[{0, j} for j in range(n)]]
    c = Case(30, [prefix], [n], 8, 2, D, 16, dtype, mode, visible=visible)
    t = prefix + big
    c.vs[int(c.bt[0, t // 16]), t % 16] *= 2.0 ** log2
    got = c.run(attn).clone()
    c.visible[0][big] = {0}  # the row that sees it is left out of the check
    ref, _, _ = c.ref()
    got[big] = ref[big].to(dtype)
    c.check(got)


@pytest.mark.parametrize("dtype,mode", [(BF16, "int8_per_token_head"), (F16, "fp8_per_token_head")])
@pytest.mark.parametrize("log2", [16, 30, 60, 100])
@pytest.mark.parametrize("at", [3, 500, 1020, 2040])
@pytest.mark.parametrize("D", [64, 128])
def test_value_scales_of_tokens_that_weigh_nothing(attn, dtype, mode, log2, at, D):
    """A token that every row sees, whose value scale is 2^log2 times the others' and whose weight
    is so small that it hardly counts: the outputs are the others' values."""
    c = Case(31, [2035], [9], 8, 2, D, 16, dtype, mode)
    page, row = int(c.bt[0, at // 16]), at % 16
    # queries of one sign, and a key against them: the score is lower by 2 log2 in the exponent of 2
    c.q = c.q.abs() * 0.05
    ones = torch.ones(c.k.shape[-1], device=DEV)
    c.k[page, row] = (-ones * (100 if mode.startswith("int8") else 240)).to(c.k.dtype)
    s = (c.q.float().sum(-1).amin() * c.scale * (100 if mode.startswith("int8") else 240)).item()
    c.ks[page, row] = 1.5 * log2 * math.log(2) / s
    c.vs[page, row] *= 2.0 ** log2
    c.check(c.run(attn))


@pytest.mark.parametrize("mode", ["int8_per_token_head", "fp8_per_token_head"])
@pytest.mark.parametrize("first,last", [(2.0 ** 60, 2.0 ** -60), (2.0 ** -60, 2.0 ** 60), (2.0 ** 30, 2.0 ** -80)])
def test_value_scales_from_tile_to_tile(attn, mode, first, last):
    """Value scales that differ by up to 2^120 between the first and the last part of the context."""
    c = Case(32, [1500, 70], [11, 3], 8, 2, 128, 16, BF16, mode)
    for b, cut in ((0, 64), (1, 2)):
        pages = c.bt[b].long()
        c.vs[pages[:cut]] *= first
        c.vs[pages[cut:-(-int(c.lens[b]) // 16)]] *= last
    c.check(c.run(attn))


@pytest.mark.parametrize("mode", ["auto", "int8_per_token_head"])
def test_replays_of_a_padded_batch_whose_trees_change(attn, mode):
    """One captured call of fixed sizes, replayed on batches of other lengths, trees and numbers of
    sequences: what was padding in one replay is a row of the next, and the other way round."""
    B, total, words = 5, 60, 1
    cases = [Case(40 + i, p, n, 8, 2, 128, 16, BF16, mode) for i, (p, n) in enumerate((
        ([50, 0, 700, 3, 9], [4, 1, 40, 10, 5]), ([1500], [3]), ([0, 20], [0, 60]), ([400, 5, 5], [1, 1, 1])))]
    NB = max(c.k.shape[0] for c in cases)
    k, v = (torch.zeros(NB, 16, 2, 128, dtype=cases[0].k.dtype, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(NB, 16, 2, device=DEV) if mode != "auto" else None for _ in range(2))
    q = torch.zeros(total, 8, 128, dtype=BF16, device=DEV)
    bt = torch.full((B, 130), -1, dtype=torch.int32, device=DEV)
    lens, cu = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    mask = torch.zeros(total, words, dtype=torch.int64, device=DEV)

    def fill(c):
        n, b = c.cu[-1], c.B
        k[:c.k.shape[0]], v[:c.k.shape[0]] = c.k, c.v
        if ks is not None:
            ks[:c.k.shape[0]], vs[:c.k.shape[0]] = c.ks, c.vs
        q[:n], q[n:] = c.q, float("nan")
        bt.fill_(-1)
        bt[:b, :c.bt.shape[1]] = c.bt
        lens.zero_(), mask.fill_(-1)
        lens[:b], mask[:n] = c.lens, c.mask
        cu[:b + 1], cu[b + 1:] = c.cut, n

    def call():
        return attn.paged_attention_tree(q, k, v, bt, lens, cu, mask, cases[0].scale, 8, 2, 128, 16, ks, vs, mode)

    fill(cases[0])
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for c in cases + cases[::-1]:
        fill(c)
        out.fill_(float("nan"))
        graph.replay()
        n = c.cu[-1]
        c.check(out[:n])
        assert (out[n:] == 0).all()
