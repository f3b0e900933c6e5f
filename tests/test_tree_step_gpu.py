"""tree_metadata, tree_accept, copy_kv_pages and move_kv_rows against plain implementations,
bit for bit, and a whole step of them with the append and the attention, eager and captured."""
import random

import pytest
import torch

from conftest import mkv_module
from oracle.tree_oracle import mask_words, paged_tree_ref, tree_accept_ref, tree_metadata_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def kv():
    return mkv_module("engine.kv_cache")


def batch(seed, nodes, prefix, BS, width=None, depth=8):
    r = random.Random(seed)
    cu, parents = [0], []
    for n in nodes:
        cu.append(cu[-1] + n)
        d = []
        for j in range(n):
            p = r.randrange(j) if j else -1
            while p >= 0 and d[p] >= depth - 1:
                p = parents[cu[-2] + p]
            parents.append(p)
            d.append(d[p] + 1 if p >= 0 else 0)
    blocks = [-(-(a + b) // BS) for a, b in zip(prefix, nodes)]
    perm = list(range(sum(blocks) + 2))
    r.shuffle(perm)
    w = width if width is not None else max(blocks + [1])
    tables, at = [], 0
    for k in blocks:
        tables.append((perm[at:at + k] + [-1] * w)[:w])
        at += k
    return cu, parents, tables


def dev(x, t=torch.int64):
    return torch.tensor(x, dtype=t, device=DEV)


@pytest.mark.parametrize("nodes,prefix,BS", [
    ([1], [0], 16), ([8], [411], 16), ([0, 5, 0, 64, 65], [3, 0, 7, 100, 9], 16), ([130, 1, 257], [1, 2, 3], 7),
    ([1024], [5], 256), ([3] * 300, list(range(300)), 16)])
@pytest.mark.parametrize("types", [(torch.int32, torch.int32, torch.int64, torch.int32),
                                   (torch.int64, torch.int64, torch.int32, torch.int64)])
def test_metadata(kv, nodes, prefix, BS, types):
    cu, parents, tables = batch(1, nodes, prefix, BS, depth=20)
    m = kv.tree_metadata(dev(parents, types[0]), dev(cu, types[1]), dev(prefix, types[2]), dev(tables, types[3]), BS,
                         max(nodes))
    words = -(-max(nodes) // 64)
    slots, lens, positions, visible = tree_metadata_ref(parents, cu, prefix, tables, BS, words)
    assert m.slot_mapping.tolist() == slots and m.context_lens.tolist() == lens
    assert m.positions.tolist() == positions
    assert torch.equal(m.tree_mask.cpu(), mask_words(visible, words))


def test_metadata_of_a_chain_of_1024(kv):
    parents = list(range(-1, 1023))
    m = kv.tree_metadata(dev(parents, torch.int32), dev([0, 1024]), dev([0]), dev([[0, 1, 2, 3]], torch.int32), 256, 1024)
    _, _, positions, visible = tree_metadata_ref(parents, [0, 1024], [0], [[0, 1, 2, 3]], 256, 16)
    assert m.positions.tolist() == positions == list(range(1024))
    assert torch.equal(m.tree_mask.cpu(), mask_words(visible, 16))


def test_metadata_of_padding_bad_parents_and_missing_pages(kv):
    """Rows behind (and before) the sequences get slot -1; a parent that is no lower node
    counts as none; a table that is too narrow, or a node past the mask, gives slot -1."""
    cu, parents, tables = [2, 6, 76], [9, 9] + [-1, 5, 1, -7] + list(range(-1, 69)) + [3, 3, 3], [[4, -1], [1, 0]]
    m = kv.tree_metadata(dev(parents, torch.int32), dev(cu), dev([14, 0]), dev(tables, torch.int32), 16, 64)
    shifted = parents[2:76]
    slots, lens, positions, visible = tree_metadata_ref(shifted, [0, 4, 74], [14, 0], tables, 16, 1)
    assert m.slot_mapping.tolist() == [-1, -1] + slots + [-1] * 3
    assert slots[:4] == [78, 79, -1, -1] and slots[4:38] == list(range(16, 32)) + list(range(0, 16)) + [-1, -1]
    assert m.context_lens.tolist() == [18, 70]
    assert m.positions.tolist() == [0, 0] + positions + [0] * 3
    want = torch.cat([torch.zeros(2, 1, dtype=torch.int64), mask_words(visible, 1), torch.zeros(3, 1, dtype=torch.int64)])
    assert torch.equal(m.tree_mask.cpu(), want)


@pytest.mark.parametrize("cu", [0, 3])
def test_metadata_of_padding_alone(kv, cu):
    """A step that is all padding (no sequence): slot -1 everywhere, so the append writes nothing."""
    m = kv.tree_metadata(dev([-1, 0, 1, 2, 0], torch.int32), dev([cu]), dev([]),
                         torch.zeros(0, 4, dtype=torch.int32, device=DEV), 16, 70)
    assert m.slot_mapping.tolist() == [-1] * 5 and m.positions.tolist() == [0] * 5
    assert m.context_lens.numel() == 0 and not m.tree_mask.any() and m.tree_mask.shape == (5, 2)


def test_prefix_past_64_bits_has_no_slots(kv):
    top = 2**63 - 1
    tables = dev([[0, 1], [1, 0]], torch.int32)
    m = kv.tree_metadata(dev([-1, 0, 0, -1], torch.int32), dev([0, 3, 4]), dev([top, 5]), tables, 16, 8)
    assert m.slot_mapping.tolist() == [-1] * 3 + [21]
    a = kv.tree_accept(dev([7, 8, 9, 7]), dev([9, 0, 0, 0]), dev([-1, 0, 0, -1], torch.int32), dev([0, 3, 4]), dev([top, 5]),
                       tables, 16, 3)
    assert a.accepted_nodes[0].tolist() == [0, 2, -1] and (a.src_slots == -1).all() and (a.dst_slots == -1).all()


@pytest.mark.parametrize("nodes", [[1], [8], [0, 5, 0, 64, 129, 300], [40] * 70])
@pytest.mark.parametrize("max_path", [1, 4, 9, 40])
@pytest.mark.parametrize("tok", [torch.int32, torch.int64])
def test_accept(kv, nodes, max_path, tok):
    r = random.Random(len(nodes) + max_path)
    prefix = [r.randrange(50) for _ in nodes]
    cu, parents, tables = batch(2, nodes, prefix, 16, depth=50)
    # few token values: siblings with equal tokens are common, the lowest index wins
    draft = [r.randrange(3) for _ in parents]
    target = [r.randrange(3) for _ in parents]
    a = kv.tree_accept(dev(draft, tok), dev(target, tok), dev(parents, torch.int32), dev(cu, torch.int32), dev(prefix),
                       dev(tables, torch.int32), 16, max_path)
    got = (a.num_accepted, a.accepted_nodes, a.tokens, a.context_lens, a.src_slots, a.dst_slots)
    want = tree_accept_ref(draft, target, parents, cu, prefix, tables, 16, max_path)
    for g, w in zip(got, want):
        assert g.tolist() == w
    if max_path == 40 and len(nodes) > 3:
        assert max(want[0]) > 4  # paths of some length are among them


def test_accept_along_a_chain_past_the_held_nodes(kv):
    n = 200
    cu, parents = [0, n], list(range(-1, n - 1))
    toks = [7 * j % 151 for j in range(n)]
    target = toks[1:] + [5]
    tables = [[2, 0, 1, 3]]
    a = kv.tree_accept(dev(toks), dev(target), dev(parents, torch.int32), dev(cu), dev([10]), dev(tables, torch.int32), 64, 256)
    assert a.num_accepted.tolist() == [n] and a.accepted_nodes[0].tolist() == list(range(n)) + [-1] * 56
    assert a.tokens[0].tolist() == target + [-1] * 56 and a.context_lens.tolist() == [10 + n]
    assert (a.src_slots == -1).all() and (a.dst_slots == -1).all()


def cache_of(kv, mode, L=3, NB=11, BS=16, KVH=2, D=64, dtype=torch.bfloat16, seed=0):
    c = kv.allocate_kv_cache(L, NB, BS, KVH, D, mode, dtype, DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    c.kv.view(torch.uint8).copy_(torch.randint(0, 256, (c.kv.numel() * c.kv.element_size(),), generator=g, device=DEV,
                                               dtype=torch.uint8).view(c.kv.view(torch.uint8).shape))
    if mode.endswith("token_head"):
        for t in (c.k_scale, c.v_scale):
            t.copy_(torch.rand(t.shape, generator=g, device=DEV))
    return c


def planes(c):
    """Every tensor that a copy touches, as bytes (planes, NB, BS, row bytes)."""
    _, L, NB, BS = c.kv.shape[:4]
    out = [c.kv.view(torch.uint8).reshape(2 * L, NB, BS, -1)]
    if c.kv_cache_dtype.endswith("token_head"):
        out += [t.view(torch.uint8).reshape(L, NB, BS, -1) for t in (c.k_scale, c.v_scale)]
    return out


def pages_ref(c, src, dst):
    for p in planes(c):
        for a, b in zip(src, dst):
            if 0 <= a < p.shape[1] and 0 <= b < p.shape[1]:
                p[:, b] = p[:, a].clone()


def rows_ref(c, src, dst):
    for p in planes(c):
        f = p.view(p.shape[0], -1, p.shape[3])
        for ga, gb in zip(src, dst):
            for a, b in zip(ga, gb):
                if 0 <= a < f.shape[1] and 0 <= b < f.shape[1]:
                    f[:, b] = f[:, a].clone()


CACHES = [("auto", torch.bfloat16, 2, 64), ("auto", torch.float32, 1, 128), ("auto", torch.float16, 3, 8),
          ("fp8_per_tensor", None, 2, 64), ("fp8_per_token_head", None, 1, 16), ("int8_per_token_head", None, 8, 128)]


@pytest.mark.parametrize("mode,dtype,KVH,D", CACHES)
@pytest.mark.parametrize("pairs", [
    [], [(3, 5)], [(0, 1), (0, 2), (0, 10)], [(1, 2), (2, 3), (3, 4), (4, 5), (5, 6), (6, 7), (7, 8), (8, 9), (9, 10)],
    [(5, 4), (4, 3), (3, 2)], [(1, 2), (3, 2), (2, 1)], [(4, 4), (-1, 3), (3, -1), (11, 2), (2, 11), (7, 8)]])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_copy_pages(kv, mode, dtype, KVH, D, pairs, index):
    """Forks, chains in either direction, pages written twice, entries that are no copies."""
    c, want = (cache_of(kv, mode, KVH=KVH, D=D, dtype=dtype or torch.bfloat16) for _ in range(2))
    src, dst = [a for a, _ in pairs], [b for _, b in pairs]
    pages_ref(want, src, dst)
    kv.copy_kv_pages(c, dev(src, index), dev(dst, index))
    for a, b in zip(planes(c), planes(want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("BS", [1, 7, 256])
@pytest.mark.parametrize("mode", ["auto", "fp8_per_token_head"])
def test_copy_pages_of_any_size_in_any_order(kv, BS, mode):
    r = random.Random(BS)
    c, want = (cache_of(kv, mode, NB=40, BS=BS, KVH=1, D=16) for _ in range(2))
    src, dst = [r.randrange(-1, 41) for _ in range(100)], [r.randrange(-1, 41) for _ in range(100)]
    pages_ref(want, src, dst)
    kv.copy_kv_pages(c, dev(src), dev(dst))
    for a, b in zip(planes(c), planes(want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("pairs", [16, 100, 700, 1024, 1025, 2500])
@pytest.mark.parametrize("kind", ["apart", "repeated source", "chained", "same destination", "self", "swapped"])
@pytest.mark.parametrize("mode", ["auto", "int8_per_token_head"])
def test_many_small_pages(kv, pairs, kind, mode):
    """Few columns and many pairs: spread over the GPU where no pair touches another's pages, in
    order where one does, in the first or the last of them."""
    NB = 2 * pairs + 5
    c, want = (cache_of(kv, mode, L=2, NB=NB, BS=2, KVH=1, D=32) for _ in range(2))
    r = random.Random(pairs)
    perm = r.sample(range(NB), NB)
    src, dst = perm[:pairs], perm[pairs:2 * pairs]
    if kind == "repeated source":
        src = [src[i // 3] for i in range(pairs)]
    elif kind == "chained":
        src[-1] = dst[0]
        src[7] = dst[6]
    elif kind == "same destination":
        dst[-1] = dst[1]
    elif kind == "self":
        dst[5], dst[9], src[11] = src[5], -1, NB
    elif kind == "swapped":  # the last one writes what the first one reads
        dst[-1] = src[0]
    pages_ref(want, src, dst)
    kv.copy_kv_pages(c, dev(src), dev(dst))
    for a, b in zip(planes(c), planes(want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("pairs", [16, 100, 1025])
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("mode", ["auto", "int8_per_token_head"])
def test_copies_onto_themselves_beside_copies_there(kv, pairs, rows, mode):
    """Padding a plan with copies of a unit onto itself changes nothing, although another pair, in
    the first or the last part of the plan, fills that unit: whatever the order of the two, the
    filled unit stays filled."""
    n = 2 * pairs + 5
    BS = 1 if rows else 2
    for first, last in ((0, pairs - 1), (pairs - 1, 0), (1, pairs // 2), (pairs // 2, 1)):
        c, want = (cache_of(kv, mode, L=2, NB=n, BS=BS, KVH=1, D=32, seed=first) for _ in range(2))
        r = random.Random(pairs + first)
        perm = r.sample(range(n), n)
        src, dst = perm[:pairs], perm[pairs:2 * pairs]
        src[first] = dst[first] = dst[last]  # onto itself, a destination of the pair `last`
        if pairs > 16:
            src[7] = dst[7] = dst[-2]
        if rows:
            rows_ref(want, [src], [dst])
        else:
            pages_ref(want, src, dst)
        for _ in range(5):  # (again: the sources are no destinations, so the result is the same)
            if rows:
                kv.move_kv_rows(c, dev([src]), dev([dst]))
            else:
                kv.copy_kv_pages(c, dev(src), dev(dst))
            for a, b in zip(planes(c), planes(want)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("mode,dtype,KVH,D", CACHES)
@pytest.mark.parametrize("G,M", [(1, 1), (1, 5), (5, 9), (11, 30), (1, 0), (0, 3)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_move_rows(kv, mode, dtype, KVH, D, G, M, index):
    """Moves within each group's own page in any order, repeated and chained; -1 padding."""
    r = random.Random(10 * G + M)
    c, want = (cache_of(kv, mode, KVH=KVH, D=D, dtype=dtype or torch.bfloat16) for _ in range(2))
    src = [[g * 16 + r.randrange(16) if r.random() < 0.9 else -1 for _ in range(M)] for g in range(G)]
    dst = [[g * 16 + r.randrange(16) if r.random() < 0.9 else -1 for _ in range(M)] for g in range(G)]
    if G == 5:
        src[2][3], dst[3][3] = 11 * 16, 1 << 30  # past the cache
    rows_ref(want, src, dst)
    kv.move_kv_rows(c, dev(src, index).reshape(G, M), dev(dst, index).reshape(G, M))
    for a, b in zip(planes(c), planes(want)):
        assert torch.equal(a, b)


def test_many_groups_and_slices(kv):
    """More groups than a grid has rows in its second dimension, from a slice of a wider table."""
    c, want = (cache_of(kv, "auto", L=1, NB=70000, BS=2, KVH=1, D=8) for _ in range(2))
    src = torch.arange(70000, device=DEV)[:, None] * 2 + torch.tensor([[0, 5]], device=DEV)
    dst = torch.arange(70000, device=DEV)[:, None] * 2 + torch.tensor([[1, 5]], device=DEV)
    kv.move_kv_rows(c, src[:, :1], dst[:, :1])
    want.kv[:, :, :, 1] = want.kv[:, :, :, 0]
    assert torch.equal(c.kv.view(torch.uint8), want.kv.view(torch.uint8))


def test_copies_past_32_bits(kv):
    """A cache of 5 GB: byte offsets beyond 32 bits in pages, rows and layers."""
    c = kv.allocate_kv_cache(2, 5000, 256, 4, 128, "auto", torch.bfloat16, DEV)
    c.kv[:, :, 4999].normal_()
    c.kv[:, :, 4998].normal_()
    page, row = c.kv[:, :, 4999].clone(), c.kv[:, :, 4998, 255].clone()
    kv.copy_kv_pages(c, dev([4999]), dev([4990]))
    kv.move_kv_rows(c, dev([[4998 * 256 + 255]]), dev([[4991 * 256]]))
    assert torch.equal(c.kv[:, :, 4990], page) and torch.equal(c.kv[:, :, 4991, 0], row)
    assert not c.kv[:, :, 4992].any() and not c.kv[:, :, 4991, 1:].any()


@pytest.mark.parametrize("mode", ["auto", "fp8_per_tensor", "fp8_per_token_head", "int8_per_token_head"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_whole_step(kv, attn, mode, captured):
    """Metadata, append, attention, acceptance and the move of the accepted rows, as a decode
    step uses them; captured, the graph is replayed on a second step's inputs. Afterwards
    the kept context holds the rows that appending the accepted tokens alone would hold."""
    r = random.Random(3)
    H, KVH, D, BS, L = 8, 2, 128, 16, 2
    nodes, prefix = [9, 20, 1, 33], [50, 0, 16, 131]
    cu, parents, tables = batch(4, nodes, prefix, BS)
    NB, total, M = 1 + max(max(t) for t in tables), cu[-1], 6
    cache = kv.allocate_kv_cache(L, NB, BS, KVH, D, mode, torch.bfloat16, DEV)
    if mode == "fp8_per_tensor":
        cache.k_scale.fill_(0.01)
        cache.v_scale.fill_(0.012)
    g = torch.Generator(device=DEV).manual_seed(5)
    norm = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    P, C, X, T = dev(parents, torch.int32), dev(cu, torch.int32), dev(prefix), dev(tables, torch.int32)
    slots = [t[i // BS] * BS + i % BS for t, n in zip(tables, prefix) for i in range(n)]

    def append(l, k, v, slot):
        kc, vc, ks, vs = cache.layer(l)
        if mode == "auto":
            attn.store_kvcache(k, v, kc, vc, slot, BS)
        elif mode == "int8_per_token_head":
            attn.store_kvcache_int8(k, v, kc, vc, ks, vs, slot, BS)
        else:
            attn.store_kvcache_fp8(k, v, kc, vc, ks, vs, slot, BS, mode)

    for l in range(L):
        append(l, norm(len(slots), KVH, D), norm(len(slots), KVH, D), dev(slots))
    start = cache.kv.clone(), None if cache.k_scale is None else (cache.k_scale.clone(), cache.v_scale.clone())
    q, k, v = norm(L, total, H, D), norm(L, total, KVH, D), norm(L, total, KVH, D)
    draft, target = dev([0] * total), dev([0] * total)

    def inputs(seed):
        rr = random.Random(seed)
        q.copy_(norm(L, total, H, D)), k.copy_(norm(L, total, KVH, D)), v.copy_(norm(L, total, KVH, D))
        d, t = [rr.randrange(900) for _ in range(total)], [rr.randrange(900) for _ in range(total)]
        depth = [0] * total
        for b, n in enumerate(nodes):  # along the way to the last of the deepest nodes the target agrees
            for j in range(1, n):
                depth[cu[b] + j] = depth[cu[b] + parents[cu[b] + j]] + 1
            j = max(range(n), key=lambda x: (depth[cu[b] + x], x))
            while j > 0:
                t[cu[b] + parents[cu[b] + j]] = d[cu[b] + j]
                j = parents[cu[b] + j]
        draft.copy_(dev(d)), target.copy_(dev(t))

    def step():
        m = kv.tree_metadata(P, C, X, T, BS, max(nodes))
        outs = []
        for l in range(L):
            append(l, k[l], v[l], m.slot_mapping)
            kc, vc, ks, vs = cache.layer(l)
            outs.append(attn.paged_attention_tree(q[l], kc, vc, T, m.context_lens, C, m.tree_mask, D ** -0.5, H, KVH, D,
                                                  BS, ks, vs, mode))
        a = kv.tree_accept(draft, target, P, C, X, T, BS, M)
        kv.move_kv_rows(cache, a.src_slots, a.dst_slots)
        return m, outs, a

    inputs(1)
    if captured:
        step()  # eagerly once, as the append asks for
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        inputs(2)
    cache.kv.view(torch.uint8).copy_(start[0].view(torch.uint8))
    if start[1] is not None:
        cache.k_scale.copy_(start[1][0]), cache.v_scale.copy_(start[1][1])
    if captured:
        graph.replay()
        m, outs, a = held
    else:
        m, outs, a = step()
    torch.cuda.synchronize()
    _, lens, _, visible = tree_metadata_ref(parents, cu, prefix, tables, BS, 1)
    want = tree_accept_ref(draft.tolist(), target.tolist(), parents, cu, prefix, tables, BS, M)
    assert a.accepted_nodes.tolist() == want[1] and a.tokens.tolist() == want[2] and max(want[0]) > 2
    after = cache.kv.clone(), None if cache.k_scale is None else (cache.k_scale.clone(), cache.v_scale.clone())
    # the kept rows are what an append of the accepted tokens alone gives
    cache.kv.view(torch.uint8).copy_(start[0].view(torch.uint8))
    if start[1] is not None:
        cache.k_scale.copy_(start[1][0]), cache.v_scale.copy_(start[1][1])
    kept = [(cu[b] + c, tables[b][(prefix[b] + i) // BS] * BS + (prefix[b] + i) % BS)
            for b in range(4) for i, c in enumerate(want[1][b]) if c >= 0]
    rows, at = dev([x for x, _ in kept]), dev([x for _, x in kept])
    for l in range(L):
        append(l, k[l][rows], v[l][rows], at)
    held_slots = dev(slots + [x for _, x in kept])
    flat = lambda x: x.view(torch.uint8).reshape(2, L, NB * BS, -1)[:, :, held_slots]  # noqa: E731
    assert torch.equal(flat(after[0]), flat(cache.kv))
    if mode.endswith("token_head"):
        for x, y in zip(after[1], (cache.k_scale, cache.v_scale)):
            assert torch.equal(x.reshape(L, NB * BS, -1)[:, held_slots], y.reshape(L, NB * BS, -1)[:, held_slots])
    # the attention saw the whole tree: the cache before the moves is the start with all nodes appended
    for l in range(L):
        append(l, k[l], v[l], m.slot_mapping)
        kc, vc, ks, vs = cache.layer(l)
        ref, mag, _ = paged_tree_ref(q[l], kc, vc, T, torch.tensor(lens), cu, visible, D ** -0.5, ks, vs)
        u = 2.0 ** -8  # outputs and weights in 16 bits: half a bf16 step each (f32 errors are far below)
        assert ((outs[l].double() - ref).abs() <= u * (ref.abs() + mag)).all()


@pytest.mark.parametrize("other", [False, True])
def test_streams(kv, other):
    """The work is queued on the current stream: behind what that stream holds."""
    s = torch.cuda.Stream() if other else torch.cuda.current_stream()
    c = cache_of(kv, "auto", L=28, NB=64)
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        for i in range(50):
            c.kv[:, :, 1].add_(0)  # work in front
        c.kv[:, :, 1] = 5
        kv.copy_kv_pages(c, dev([1]), dev([2]))
        kv.move_kv_rows(c, dev([[2 * 16 + 1]]), dev([[3 * 16]]))
        got = c.kv.clone()
    s.synchronize()
    assert (got[:, :, 2] == 5).all() and (got[:, :, 3, 0] == 5).all()


def test_c_entry_points_and_their_counts(kv):
    """The C calls themselves (the wrappers make them packed): the same results, and the entries
    that they skip are counted."""
    lib_mod = mkv_module("_lib")
    lib = lib_mod.load()
    I32, I64 = lib_mod.INDEX_I32, lib_mod.INDEX_I64
    stream = torch.cuda.current_stream().cuda_stream
    bad = dev([0], torch.int32)
    par, cu, pre, bt = dev([-1, 0, 5, -3, 1], torch.int32), dev([0, 3, 5]), dev([4, 9]), dev([[3, 1], [2, 0]], torch.int32)
    outs = [torch.empty(n, dtype=torch.int64, device=DEV) for n in (5, 2, 5, 5)]
    st = lib.mkv_tree_metadata(par.data_ptr(), I32, cu.data_ptr(), I64, pre.data_ptr(), I64, bt.data_ptr(), I32, 2, 2, 8, 2,
                               5, 1, *[o.data_ptr() for o in outs], bad.data_ptr(), stream)
    lib_mod.check("mkv_tree_metadata", st)
    m = kv.tree_metadata(par, cu, pre, bt, 8, 3)
    for a, b in zip(outs, (m.slot_mapping, m.context_lens, m.positions, m.tree_mask.view(-1))):
        assert torch.equal(a, b)
    assert bad.tolist() == [3]  # the parents 5, -3 and 1 (of node 1: not a lower one)
    draft, target = dev([7, 8, 9, 1, 2]), dev([8, 4, 5, 6, 3])
    par = dev([-1, 0, 0, -1, 0], torch.int32)
    wide = [torch.empty(2, 4, dtype=torch.int64, device=DEV) for _ in range(3)]
    nodes, count = torch.empty(2, 4, dtype=torch.int32, device=DEV), dev([0, 0], torch.int32)
    lens = dev([0, 0])
    st = lib.mkv_tree_accept(draft.data_ptr(), target.data_ptr(), I64, par.data_ptr(), I32, cu.data_ptr(), I64,
                             pre.data_ptr(), I64, bt.data_ptr(), I32, 2, 2, 8, 2, 5, 4, count.data_ptr(), nodes.data_ptr(),
                             wide[0].data_ptr(), lens.data_ptr(), wide[1].data_ptr(), wide[2].data_ptr(), stream)
    lib_mod.check("mkv_tree_accept", st)
    a = kv.tree_accept(draft, target, par, cu, pre, bt, 8, 4)
    for x, y in zip([count, nodes, lens] + wide, (a.num_accepted, a.accepted_nodes, a.context_lens, a.tokens, a.src_slots,
                                                  a.dst_slots)):
        assert torch.equal(x, y)
    for split in (False, True):  # a few pairs, and so many that they are spread over the GPU
        c, want = (cache_of(kv, "int8_per_token_head", L=2, NB=70, BS=2, KVH=1, D=32) for _ in range(2))
        src, dst = ([3, -1, 70, 5, 9], [4, 2, 6, 1 << 40, 9]) if not split else \
            ([3, -1, 70, 5, 9] + list(range(10, 40)), [4, 2, 6, 1 << 40, 8] + list(range(40, 70)))
        pages_ref(want, src, dst)
        bad.zero_()
        s, d = dev(src), dev(dst)
        k = c.kv.data_ptr()
        st = lib.mkv_copy_kv_pages(k, k + c.kv.numel() // 2, lib_mod.DTYPE_INT8, 2, 70 * 2 * 32, 70, 2, 1, 32,
                                   c.k_scale.data_ptr(), c.v_scale.data_ptr(), 140, s.data_ptr(), d.data_ptr(), I64, len(src),
                                   bad.data_ptr(), stream)
        lib_mod.check("mkv_copy_kv_pages", st)
        for x, y in zip(planes(c), planes(want)):
            assert torch.equal(x, y)
        assert bad.tolist() == [2]
    rows_ref(want, [[1, 140, 2]], [[0, 3, 5]])
    bad.zero_()
    s, d = dev([[1, 140, 2]]), dev([[0, 3, 5]])
    st = lib.mkv_move_kv_rows(k, k + c.kv.numel() // 2, lib_mod.DTYPE_INT8, 2, 70 * 2 * 32, 70, 2, 1, 32,
                              c.k_scale.data_ptr(), c.v_scale.data_ptr(), 140, s.data_ptr(), d.data_ptr(), I64, 1, 3,
                              bad.data_ptr(), stream)
    lib_mod.check("mkv_move_kv_rows", st)
    for x, y in zip(planes(c), planes(want)):
        assert torch.equal(x, y)
    assert bad.tolist() == [1]


def test_packed_calls_refuse():
    lib_mod = mkv_module("_lib")
    lib = lib_mod.load()
    assert lib.mkv_call_packed(5, b"\0" * 400) == 1 and b"unknown call" in lib.mkv_last_error()
    assert lib.mkv_call_packed(0, None) == 1 and b"null pointer" in lib.mkv_last_error()


def test_invalid_entries_are_counted(kv):
    """Trees that are none, trees wider than their masks, and copies past the cache can be noticed
    through the public functions; the results are those without the count."""
    bad = dev([5], torch.int32)  # it is added to
    parents, cu = [-1, 0, 7, 1, -9] + list(range(-1, 69)), [0, 5, 75]
    args = (dev(parents, torch.int32), dev(cu), dev([3, 0]), dev([[4, 1], [3, 2]], torch.int32), 16)
    a, b = kv.tree_metadata(*args, 64), kv.tree_metadata(*args, 64, invalid_count=bad)
    assert bad.tolist() == [5 + 2 + 6]  # parents 7 and -9; nodes 64 to 69
    for x, y in zip((a.slot_mapping, a.context_lens, a.positions, a.tree_mask),
                    (b.slot_mapping, b.context_lens, b.positions, b.tree_mask)):
        assert torch.equal(x, y)
    kv.tree_metadata(*args, 70, invalid_count=bad)
    assert bad.tolist() == [15]
    c, want = (cache_of(kv, "auto") for _ in range(2))
    pages_ref(want, [1, 11, 3, -1], [2, 4, 1 << 20, 5])
    kv.copy_kv_pages(c, dev([1, 11, 3, -1]), dev([2, 4, 1 << 20, 5]), invalid_count=bad.zero_())
    assert bad.tolist() == [2]
    rows_ref(want, [[1, -1], [176, 7]], [[0, 3], [5, 8]])
    kv.move_kv_rows(c, dev([[1, -1], [176, 7]]), dev([[0, 3], [5, 8]]), invalid_count=bad)
    assert bad.tolist() == [3]
    assert torch.equal(planes(c)[0], planes(want)[0])
    with pytest.raises(ValueError, match="invalid_count"):
        kv.copy_kv_pages(c, dev([1]), dev([2]), invalid_count=torch.zeros(1, dtype=torch.int32))
