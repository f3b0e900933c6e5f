"""Refusals of the tree and cache-copy entry points, through the C ABI and the wrappers; no
call here reaches a CUDA API."""
import pytest
import torch

from conftest import mkv_module

lib_mod = mkv_module("_lib")
kv = mkv_module("engine.kv_cache")
P = 1 << 20  # a pointer that nothing reads


def _tree(lib, **kw):
    a = dict(q=P, qst=1024, qsh=128, qdt=2, k=P, v=P, cdt=2, ks=None, vs=None, kss=None, vss=None, nb=10, bs=16, bt=P,
             btt=0, btst=8, maxb=8, cl=P, clt=1, cu=P, cut=0, mask=P, mst=1, words=1, B=2, T=9, H=8, KVH=2, D=128,
             scale=0.1, out=P, ost=1024, osh=128, ws=P, wsb=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.mkv_paged_tree_attention(*a.values())


@pytest.mark.parametrize("kw,status,msg", [
    (dict(H=7), 1, b"multiple of num_kv_heads"),
    (dict(D=100), 2, b"head_dim"),
    (dict(D=272), 2, b"head_dim"),
    (dict(qdt=3), 2, b"query dtype"),
    (dict(cdt=1), 2, b"cache dtype"),
    (dict(cdt=3), 1, b"needs k_scale and v_scale"),
    (dict(cdt=3, ks=P), 1, b"needs k_scale and v_scale"),
    (dict(cdt=3, ks=P, vs=P, kss=P, vss=P), 1, b"needs k_scale and v_scale"),
    (dict(cdt=4, ks=P, vs=P), 1, b"INT8"),
    (dict(ks=P, vs=P), 1, b"unquantised"),
    (dict(btt=2), 1, b"index types"),
    (dict(clt=-1), 1, b"index types"),
    (dict(cut=9), 1, b"index types"),
    (dict(words=0), 1, b"bad sizes"),
    (dict(bs=0), 1, b"bad sizes"),
    (dict(B=-1), 1, b"bad sizes"),
    (dict(q=None), 1, b"null pointer"),
    (dict(mask=None), 1, b"null pointer"),
    (dict(bt=None), 1, b"null pointer"),
    (dict(k=P + 8), 1, b"16-byte aligned"),
    (dict(ws=None), 3, b"workspace"),
    (dict(wsb=1000), 3, b"workspace"),
    (dict(ws=P + 4), 3, b"workspace"),
    (dict(maxb=1 << 28), 2, b"2^31 tokens"),
    (dict(T=1 << 40), 2, b"2^31"),
])
def test_attention_refusals(kw, status, msg):
    lib = lib_mod.load()
    assert _tree(lib, **kw) == status
    assert msg in lib.mkv_last_error()


def test_nothing_to_do():
    lib = lib_mod.load()
    assert _tree(lib, B=0, q=None, out=None, ws=None, wsb=0) == 0
    assert _tree(lib, T=0, q=None, out=None, ws=None, wsb=0) == 0
    assert lib.mkv_paged_tree_workspace_bytes(0, 5, 8, 2, 128, 2, 2) == 0
    assert lib.mkv_paged_tree_workspace_bytes(2, 9, 8, 2, 128, 2, 2) > 0
    assert lib.mkv_tree_metadata(None, 0, None, 0, None, 0, None, 0, 0, 0, 16, 0, 0, 1, None, None, None, None, None,
                                 None) == 0
    assert lib.mkv_copy_kv_pages(None, None, 2, 4, 0, 10, 16, 2, 128, None, None, 0, None, None, 0, 0, None, None) == 0
    assert lib.mkv_move_kv_rows(None, None, 2, 4, 0, 10, 16, 2, 128, None, None, 0, None, None, 0, 3, 0, None, None) == 0


@pytest.mark.parametrize("kw,status,msg", [
    (dict(pt=7), 1, b"index types"), (dict(words=0), 2, b"mask_words"), (dict(words=17), 2, b"mask_words"),
    (dict(bs=0), 1, b"bad sizes"), (dict(B=-2), 1, b"bad sizes"), (dict(cu=None), 1, b"null pointer"),
    (dict(slots=None), 1, b"null output"), (dict(bt=None), 1, b"null pointer"),
    (dict(B=0, cu=None), 1, b"null pointer"), (dict(B=0, slots=None), 1, b"null output")])
def test_metadata_refusals(kw, status, msg):
    a = dict(par=P, pt=0, cu=P, ct=0, pre=P, prt=1, bt=P, btt=0, bts=4, maxb=4, bs=16, B=2, T=5, words=1, slots=P, lens=P,
             pos=P, mask=P, bad=None, stream=None)
    a.update(kw)
    lib = lib_mod.load()
    assert lib.mkv_tree_metadata(*a.values()) == status
    assert msg in lib.mkv_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(tt=3), 1, b"token_index_type"), (dict(path=0), 1, b"max_path"), (dict(draft=None), 1, b"null pointer"),
    (dict(dst=None), 1, b"null pointer"), (dict(T=-1), 1, b"bad sizes")])
def test_accept_refusals(kw, status, msg):
    a = dict(draft=P, target=P, tt=1, par=P, pt=0, cu=P, ct=0, pre=P, prt=1, bt=P, btt=0, bts=4, maxb=4, bs=16, B=2, T=5,
             path=3, count=P, nodes=P, tokens=P, lens=P, src=P, dst=P, stream=None)
    a.update(kw)
    lib = lib_mod.load()
    assert lib.mkv_tree_accept(*a.values()) == status
    assert msg in lib.mkv_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(cdt=7), 2, b"cache dtype"), (dict(D=4, KVH=1), 2, b"multiple of 16"), (dict(it=4), 1, b"index_type"),
    (dict(ks=P), 1, b"both"), (dict(k=P + 8), 1, b"16-byte aligned"), (dict(ls=4), 1, b"16-byte aligned"),
    (dict(ks=P + 2, vs=P), 1, b"4-byte aligned"), (dict(src=None), 1, b"null pointer"), (dict(NB=-1), 1, b"bad sizes"),
    (dict(n=1 << 40), 1, b"bad sizes")])
def test_copy_refusals(kw, status, msg):
    a = dict(k=P, v=P, cdt=2, L=2, ls=40960, NB=10, BS=16, KVH=2, D=128, ks=None, vs=None, ss=0, src=P, dst=P, it=1, n=3,
             bad=None, stream=None)
    a.update(kw)
    lib = lib_mod.load()
    assert lib.mkv_copy_kv_pages(*a.values()) == status
    assert msg in lib.mkv_last_error()


def test_wrappers_refuse(attn):
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    c = torch.zeros(8, 16, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    bt, cu, mask = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([0, 3]), torch.zeros(3, 1, dtype=torch.int64)
    args = (c, c, bt, i, cu, mask, 0.1, 8, 2, 128, 16)
    with pytest.raises(ValueError, match="CUDA"):
        attn.paged_attention_tree(q, *args)
    with pytest.raises(ValueError, match="query must be"):
        attn.paged_attention_tree(q[:, :4], *args)
    with pytest.raises(ValueError, match="query dtype"):
        attn.paged_attention_tree(q.double(), *args)
    with pytest.raises(NotImplementedError, match="kivi"):
        attn.paged_attention_tree(q, *args, None, None, "kivi_2bit")
    with pytest.raises(ValueError, match="needs k_scale"):
        attn.paged_attention_tree(q, *args, None, None, "fp8_per_tensor")
    with pytest.raises(ValueError, match="out must"):
        attn.paged_attention_tree(q, *args, out=torch.zeros(3, 8, 128))
    par = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kv.tree_metadata(par, cu, i, bt, 16, 8)
    with pytest.raises(ValueError, match="max_nodes"):
        kv.tree_metadata(par, cu, i, bt, 16, 1025)
    with pytest.raises(ValueError, match="CUDA"):
        kv.tree_accept(par.long(), par.long(), par, cu, i, bt, 16, 4)
    cache = kv.allocate_kv_cache(2, 4, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        kv.copy_kv_pages(cache, par, par)
    with pytest.raises(ValueError, match="CUDA"):
        kv.move_kv_rows(cache, par.view(1, 3), par.view(1, 3))


def test_packed_calls_are_the_calls():
    """mkv_call_packed passes each word to the parameter it stands for: refusals come out of the
    same argument, whichever way the call is made."""
    lib = lib_mod.load()
    words = dict(q=P, qst=1024, qsh=128, qdt=2, k=P, v=P, cdt=2, ks=0, vs=0, kss=0, vss=0, nb=10, bs=16, bt=P, btt=0,
                 btst=8, maxb=8, cl=P, clt=1, cu=P, cut=0, mask=P, mst=1, words=1, B=2, T=9, H=8, KVH=2, D=128, scale=0.1,
                 out=P, ost=1024, osh=128, ws=P, wsb=1 << 40, stream=0)
    for kw in (dict(H=7), dict(D=100), dict(qdt=3), dict(cdt=4), dict(btt=2), dict(clt=5), dict(cut=9), dict(words=0),
               dict(bs=0), dict(mask=0), dict(out=0), dict(k=P + 8), dict(wsb=10), dict(ws=P + 4), dict(maxb=1 << 28)):
        got = lib.mkv_call_packed(lib_mod.CALL_PAGED_TREE_ATTENTION, lib_mod.PACK_TREE_ATTENTION(*{**words, **kw}.values()))
        message = lib.mkv_last_error()
        null = {n: v or None for n, v in kw.items() if n in ("mask", "out")}
        assert got == _tree(lib, **{**kw, **null}) != 0 and message == lib.mkv_last_error()
    for call, pack, n in ((lib_mod.CALL_TREE_METADATA, lib_mod.PACK_TREE_METADATA, 20),
                          (lib_mod.CALL_TREE_ACCEPT, lib_mod.PACK_TREE_ACCEPT, 24),
                          (lib_mod.CALL_COPY_KV_PAGES, lib_mod.PACK_COPY_PAGES, 18),
                          (lib_mod.CALL_MOVE_KV_ROWS, lib_mod.PACK_MOVE_ROWS, 19)):
        assert lib.mkv_call_packed(call, pack(*[-1] * n)) != 0


def test_the_oracle_itself():
    """The plain implementations on an example worked out by hand."""
    from oracle.tree_oracle import mask_words, tree_accept_ref, tree_metadata_ref
    parents, cu, tables = [-1, 0, 0, 2, 2], [0, 5], [[7, 4]]
    slots, lens, positions, visible = tree_metadata_ref(parents, cu, [14], tables, 16, 1)
    assert slots == [126, 127, 64, 65, 66] and lens == [19] and positions == [14, 15, 15, 16, 16]
    assert mask_words(visible, 1).tolist() == [[1], [3], [5], [13], [21]]
    got = tree_accept_ref([9, 5, 6, 8, 8], [6, 1, 8, 2, 3], parents, cu, [14], tables, 16, 4)
    assert got == ([3], [[0, 2, 3, -1]], [[6, 8, 2, -1]], [17], [[-1, 64, 65, -1]], [[-1, 127, 64, -1]])


def test_the_roles_of_a_kernel_meet_at_bounded_barriers_only():
    """A warp that gives up a wait leaves its loop. What the others wait for then has to have a
    limit: no barrier over a part of the threads (bar / barrier with a number of its own), and no
    loop on an mbarrier but the one in mbar_wait, which counts the clocks."""
    import pathlib
    import re
    csrc = pathlib.Path(lib_mod.PKG_DIR) / "csrc"
    files = sorted(csrc.glob("*.cu*"))
    assert files
    for f in files:
        code = re.sub(r"//[^\n]*", "", f.read_text())
        assert not re.search(r"\b(bar|barrier)(\.cta)?\.(sync|red|arrive)", code), f.name
        assert not re.search(r"__barrier_sync|named_barrier|cuda::barrier", code), f.name
        waits = [m.start() for m in re.finditer(r"mbarrier\.try_wait|mbarrier\.test_wait", code)]
        assert len(waits) == (1 if f.name == "sm100.cuh" else 0), f.name


def test_the_zeroed_variant_refuses_the_same():
    """mkv_paged_tree_attention_zeroed, and the packed call of it."""
    lib = lib_mod.load()
    words = dict(q=P, qst=1024, qsh=128, qdt=2, k=P, v=P, cdt=2, ks=0, vs=0, kss=0, vss=0, nb=10, bs=16, bt=P, btt=0,
                 btst=8, maxb=8, cl=P, clt=1, cu=P, cut=0, mask=P, mst=1, words=1, B=2, T=9, H=8, KVH=2, D=128, scale=0.1,
                 out=P, ost=1024, osh=128, ws=P, wsb=1 << 40, stream=0)
    for kw, status in ((dict(H=7), 1), (dict(D=100), 2), (dict(mask=0), 1), (dict(out=0), 1), (dict(B=0, out=0), 1),
                       (dict(wsb=10), 3), (dict(B=0, k=P + 8), 1), (dict(T=0, out=0), 0)):
        a = {**words, **kw}
        packed = lib.mkv_call_packed(lib_mod.CALL_PAGED_TREE_ATTENTION + lib_mod.CALL_ZEROED,
                                     lib_mod.PACK_TREE_ATTENTION(*a.values()))
        message = lib.mkv_last_error()
        assert packed == lib.mkv_paged_tree_attention_zeroed(*[v or None if type(v) is int and n in (
            "q", "k", "v", "ks", "vs", "kss", "vss", "bt", "cl", "cu", "mask", "out", "ws", "stream") else v
            for n, v in a.items()]) == status
        assert message == lib.mkv_last_error() and (status == 0 or b"mkv_paged_tree_attention_zeroed" in message)
    assert lib.mkv_call_packed(lib_mod.CALL_MOVE_KV_ROWS + lib_mod.CALL_ZEROED, b"\0" * 400) == 1


def test_the_limit_of_waits():
    lib = lib_mod.load()
    first = lib.mkv_set_wait_limit(123)
    assert first == 2_000_000_000
    assert lib.mkv_set_wait_limit(-5) == 123  # below 0 counts as 0
    assert lib.mkv_set_wait_limit(first) == 0
    assert lib.mkv_set_wait_limit(first) == first


def test_tables_near_2_31_tokens():
    """Indices of tokens are 32-bit in the kernels, which look up to three tiles of 128 past the tile
    that holds the last token: a table must end 128 + 3 * 128 tokens before 2^31 at the least."""
    lib = lib_mod.load()
    for blocks, bs in (((1 << 31) // 256 - 2, 256), ((1 << 31) // 8 - 65, 8), ((1 << 31) - 512, 1), ((1 << 31) - 1023, 1)):
        assert _tree(lib, maxb=blocks, bs=bs, wsb=1000) == 2 and b"2^31 tokens" in lib.mkv_last_error()
    for blocks, bs in (((1 << 31) // 256 - 4, 256), ((1 << 31) - 1024, 1)):  # past this check, on to the next one
        assert _tree(lib, maxb=blocks, bs=bs, wsb=1000) == 3
        last = blocks * bs - 1
        assert (last // 128 + 1) * 128 - 1 + 3 * 128 < 2 ** 31


def test_counts_are_one_int32_on_the_device():
    one = torch.zeros(1, dtype=torch.int32)
    assert kv._count("f", None, 0) == 0 and kv._count("f", one, -1) == one.data_ptr()
    for t, idx in ((one, 0), (one.long(), -1), (torch.zeros(2, dtype=torch.int32), -1)):
        with pytest.raises(ValueError, match="invalid_count"):
            kv._count("f", t, idx)


@pytest.mark.parametrize("size", [0, -16, 1 << 31, (1 << 32) + 16])
def test_sizes_that_do_not_fit_the_c_call(size):
    """They are refused, not cut to 32 bits ((1 << 32) + 16 would be read as 16)."""
    par, cu, pre, bt = torch.zeros(3, dtype=torch.int32), torch.tensor([0, 3]), torch.tensor([4]), torch.zeros(1, 4).int()
    with pytest.raises(ValueError, match="block_size"):
        kv._tree_args("f", par, cu, pre, bt, size)
    with pytest.raises(ValueError, match="max_path"):
        kv.tree_accept(par, par, par, cu, pre, bt, 16, size)


def test_loads_in_flight_are_waited_for_whoever_gives_up():
    """A block whose wait has run out uses its shared memory again, so no load may still be on its way
    there: the producer's last waits do not ask whether anyone has given up (another warp may do so
    later), and the issuer of the products waits for them the same way."""
    import pathlib
    import re
    code = (pathlib.Path(lib_mod.PKG_DIR) / "csrc" / "paged_tree_tc.cu").read_text()
    for what in (r"mbar_wait\(&rfull\[k % kRS\], \(k / kRS\) & 1, nullptr\)", r"mbar_wait\(&kfull\[k % kKS\], \(k / kKS\) & 1, nullptr\)",
                 r"mbar_wait\(&vfull\[k % kVS\], \(k / kVS\) & 1, nullptr\)", r"mbar_wait\(drain, 0, nullptr\)"):
        at = [m.start() for m in re.finditer(what, code)]
        assert len(at) == 1, what
        guards = re.findall(r"if \(([^{};]*)\) \{", code[code.rindex("if (!ok) *abort_flag = 1;", 0, at[0]):at[0]])
        assert guards and not any("abort" in g for g in guards), guards
