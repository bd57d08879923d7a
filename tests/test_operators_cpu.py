"""What the rotary, 8-bit and block-attention entry points refuse: the Python checks on CPU tensors, the C checks with pointers that
are never followed (a refused call launches nothing)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def sitk_mods():
    import sitk  # noqa: F401
    from sitk import ops, runtime
    return ops, runtime


def refused(rt, fn, text):
    with pytest.raises(rt.SitkError, match=text):
        fn()


def test_rope_refusals(sitk_mods):
    ops, rt = sitk_mods
    q, k = torch.zeros(2, 5, 3, 16), torch.zeros(2, 5, 1, 16)
    pos, f = torch.zeros(5, 2), ops.rope_freqs((4, 4), device="cpu")
    ok = dict(positions=pos, freqs=f, sections=(4, 4))

    def call(**kw):
        a = dict(dict(q=q, k=k, **ok), **kw)
        return lambda: ops.rope_axes(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("freqs"), a.pop("sections"), **a)

    refused(rt, call(), "must live on a ROCm/HIP device")
    refused(rt, call(q=q.double()), "unsupported type")
    refused(rt, call(k=k.half()), "one type")
    refused(rt, call(q=q[0]), "B, N, H, dh")
    refused(rt, call(k=torch.zeros(2, 4, 1, 16)), "belong together")
    refused(rt, call(sections=(8, 4)), "do not fit")
    refused(rt, call(sections=(9, -1)), "do not fit")
    refused(rt, call(sections=(1, 1, 1, 1, 1)), "1 to 4")
    refused(rt, call(positions=torch.zeros(5, 3)), "positions")
    refused(rt, call(positions=torch.zeros(5, 2, dtype=torch.float16)), "positions of type")
    refused(rt, call(freqs=f.float()), "64-bit")
    refused(rt, call(freqs=f[:5]), "64-bit")
    refused(rt, call(q=torch.zeros(2, 5, 16, 3).transpose(2, 3)), "contiguous")
    refused(rt, call(q=q[:1].expand(2, 5, 3, 16), inplace=True), "broadcast")
    refused(rt, call(k=q, inplace=True), "share features")
    refused(rt, call(k=q[:, :, :1], inplace=True), "share features")
    both = torch.zeros(2, 5, 4, 16)
    refused(rt, call(q=both[:, :, :3], k=both[:, :, 2:], inplace=True), "share features")
    wide = torch.zeros(2, 5, 3, 2, 32)                         # apart: q and k side by side, head by head
    refused(rt, call(q=wide[:, :, :, 0, :16], k=wide[:, :, :, 1, :16], inplace=True), "must live on a ROCm/HIP device")
    refused(rt, call(q=wide[:, :, :, 0, :16], k=wide[:, :, :, 0, 8:24], inplace=True), "share features")
    refused(rt, call(q=both[:, :, :3], k=both[:, :, 3:], inplace=True), "must live on a ROCm/HIP device")


def test_rope_c_refusals(sitk_mods):
    _, rt = sitk_mods
    t = (rt.RopeTensor * 1)(rt.RopeTensor(16, 16, 2, 64, 32, 16, 64, 32, 16))
    sec = (C.c_int * 2)(4, 4)

    def rc(t=t, count=1, pos=16, kind=0, freqs=16, sec=sec, axes=2, B=1, N=2, dh=16, dtype=1):
        return rt.lib.sitk_rope_axes(t, count, pos, kind, 0, 2, freqs, sec, axes, B, N, dh, 0, 0, dtype, None)

    for kw in (dict(t=None), dict(count=3), dict(pos=None), dict(freqs=None), dict(kind=4), dict(axes=5), dict(axes=0), dict(B=-1),
               dict(dh=15), dict(dtype=9), dict(sec=(C.c_int * 2)(0, 0)), dict(sec=(C.c_int * 2)(-1, 4)),
               dict(t=(rt.RopeTensor * 1)(rt.RopeTensor(16, None, 2))), dict(B=1 << 30, N=1 << 20)):
        assert rc(**kw) == -1, kw
        assert rt.lib.sitk_last_error()
    assert rc(B=0) == 0 and rc(N=0) == 0


def test_act8_refusals(sitk_mods):
    ops, rt = sitk_mods
    refused(rt, lambda: ops.act8_pack(torch.zeros(3, 32)), "must live on")
    refused(rt, lambda: ops.act8_pack(torch.zeros(3, 32, dtype=torch.int32)), "unsupported type")
    refused(rt, lambda: ops.act8_pack(torch.zeros(())), "at least one feature")
    refused(rt, lambda: ops.act8_pack(torch.zeros(3, 0)), "at least one feature")
    p = ops.Packed8(torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.uint8), (3, 40), torch.bfloat16)
    refused(rt, lambda: ops.act8_unpack(p), "must live on")
    refused(rt, lambda: ops.act8_unpack(p, out=torch.zeros(3, 40)), "contiguous")
    refused(rt, lambda: ops.act8_gelu_bwd(torch.zeros(3, 41, dtype=torch.bfloat16), p), "does not belong")
    refused(rt, lambda: ops.act8_wgrad(torch.zeros(3, 8), p), "the rows were")
    refused(rt, lambda: ops.act8_wgrad(torch.zeros(4, 8, dtype=torch.bfloat16), p), "rows of dY")
    refused(rt, lambda: ops.act8_wgrad(torch.zeros(3, 8, dtype=torch.bfloat16), p, db=torch.zeros(8)), "db without dW")
    refused(rt, lambda: ops.act8_wgrad(torch.zeros(3, 8, dtype=torch.bfloat16), p, dW=torch.zeros(8, 41)), "dW must be")
    refused(rt, lambda: ops.act8_wgrad(torch.zeros(3, 8, dtype=torch.bfloat16), p, dW=torch.zeros(8, 40), db=torch.zeros(7)), "db must be")


def test_act8_c_refusals(sitk_mods):
    _, rt = sitk_mods
    L = rt.lib
    assert L.sitk_act8_code_bytes(3, 33) == 192 and L.sitk_act8_step_bytes(3, 33) == 6 and L.sitk_act8_code_bytes(3, 0) == 0
    assert L.sitk_act8_pack(None, 32, 16, 16, 3, 32, 1, None) == -1
    assert L.sitk_act8_pack(16, 31, 16, 16, 3, 32, 1, None) == -1
    assert L.sitk_act8_pack(16, 32, 16, 16, 3, 32, 7, None) == -1
    assert L.sitk_act8_pack(16, 32, 16, 16, -1, 32, 1, None) == -1
    assert L.sitk_act8_pack(16, 32, 16, 16, 1 << 40, 32, 1, None) == -1
    assert L.sitk_act8_pack(16, 32, 16, 16, 0, 32, 1, None) == 0
    assert L.sitk_act8_unpack(16, 16, None, 32, 3, 32, 1, None) == -1
    assert L.sitk_act8_gelu_fwd(16, 32, None, 32, 16, 16, 3, 32, 1, None) == -1
    assert L.sitk_act8_gelu_bwd(16, 32, 16, 16, 16, 8, 3, 32, 1, None) == -1
    need = L.sitk_act8_wgrad_ws_bytes(40000, 64, 64, 1)
    assert need > 0
    assert L.sitk_act8_wgrad(16, 64, 16, 16, 16, 64, 16, 40000, 64, 64, 0, 16, need - 1, 1, None) == -1
    assert L.sitk_act8_wgrad(16, 64, 16, 16, 16, 64, 16, 40000, 64, 64, 0, None, need, 1, None) == -1
    assert L.sitk_act8_wgrad(16, 63, 16, 16, 16, 64, 16, 40, 64, 64, 0, 16, need, 1, None) == -1
    assert L.sitk_act8_wgrad(16, 64, 16, 16, 16, 63, 16, 40, 64, 64, 0, 16, need, 1, None) == -1
    assert L.sitk_act8_wgrad(None, 64, 16, 16, 16, 64, 16, 40, 64, 64, 0, 16, need, 1, None) == -1
    assert L.sitk_act8_wgrad(16, 64, 16, 16, 16, 64, 16, 1 << 31, 64, 64, 0, 16, need, 1, None) == -1


def test_block_refusals(sitk_mods):
    ops, rt = sitk_mods
    k = torch.zeros(2, 300, 2, 64)
    q = torch.zeros(2, 10, 4, 64)
    refused(rt, lambda: ops.block_pool(k, 64), "must live on")
    refused(rt, lambda: ops.block_pool(k, 65), "multiple of 64")
    refused(rt, lambda: ops.block_pool(k, 0), "multiple of 64")
    refused(rt, lambda: ops.block_pool(k, 2048), "at most 1024")
    refused(rt, lambda: ops.block_pool(k[..., :32], 64), "heads, 64")
    refused(rt, lambda: ops.block_pool(k.double(), 64), "unsupported type")
    refused(rt, lambda: ops.block_pool(k, 64, key_mask=torch.ones(2, 299, dtype=torch.bool)), "key_mask")
    refused(rt, lambda: ops.block_pool(k, 64, key_mask=torch.ones(2, 300)), "key_mask")
    pool = ops.BlockPool(torch.zeros(1 << 16, dtype=torch.uint8), 2, 300, 2, 64, torch.float32)
    refused(rt, lambda: ops.block_select(q, pool, 2), "must live on")
    refused(rt, lambda: ops.block_select(q, pool, 0), "top_k")
    refused(rt, lambda: ops.block_select(q[:1], pool, 2), "does not belong")
    refused(rt, lambda: ops.block_select(q[:, :, :3], pool, 2), "does not belong")
    refused(rt, lambda: ops.block_select(q.half(), pool, 2), "does not belong")
    refused(rt, lambda: ops.block_selection(torch.zeros(2, 4, 10, 3), pool), "index of type")
    refused(rt, lambda: ops.block_selection(torch.zeros(2, 3, 10, 3, dtype=torch.int32), pool), "index must be")
    refused(rt, lambda: ops.block_selection(torch.zeros(2, 4, 10, 3, dtype=torch.int32), pool), "must live on")
    sel = ops.BlockSelection(torch.zeros(2, 4, 10, 3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), pool)
    refused(rt, lambda: ops.block_attention_fwd(q, k, k, sel, 0.125), "must live on")
    refused(rt, lambda: ops.block_attention_fwd(q, k, k, sel, 0.0), "scale")
    refused(rt, lambda: ops.block_attention_fwd(q, k, k, sel, float("nan")), "scale")
    refused(rt, lambda: ops.block_attention_fwd(q, k, k.half(), sel, 0.125), "one type")
    refused(rt, lambda: ops.block_attention_fwd(q[:, :9], k, k, sel, 0.125), "does not belong")
    refused(rt, lambda: ops.block_attention_fwd(q, k[:, :299], k, sel, 0.125), "does not belong")
    lse = torch.zeros(2, 4, 10)
    refused(rt, lambda: ops.block_attention_bwd(q, k, k, q, q[:, :9], lse, sel, 0.125), "not like q")
    refused(rt, lambda: ops.block_attention_bwd(q, k, k, q, q, lse[:1], sel, 0.125), "must be what")


def test_block_c_refusals(sitk_mods):
    _, rt = sitk_mods
    L = rt.lib
    rows = rt.BlockRows(0, 64, 64)
    byref = C.byref

    def pool(k=16, ks=byref(rows), pooled=16, B=1, Nk=100, Hk=1, block=64, dtype=1):
        return L.sitk_block_pool(k, ks, None, 0, pooled, B, Nk, Hk, block, dtype, None)

    for kw in (dict(k=None), dict(k=8), dict(ks=None), dict(ks=byref(rt.BlockRows(0, 65, 64))), dict(pooled=None), dict(B=0), dict(Nk=0),
               dict(block=63), dict(block=96), dict(block=1088), dict(dtype=5), dict(Nk=64 * 2048 + 1), dict(Nk=1024 * 300, block=1024), dict(B=1 << 20, Nk=64 * 2048)):
        assert pool(**kw) == -1 and L.sitk_last_error(), kw

    def select(q=16, H=4, Hk=2, top_k=3, index=16, Nq=10):
        return L.sitk_block_select(q, byref(rows), 16, index, 16, 1, Nq, 100, H, Hk, 64, top_k, 1, None)

    for kw in (dict(q=None), dict(H=3), dict(top_k=0), dict(index=None), dict(Nq=0), dict(Nq=1 << 30)):
        assert select(**kw) == -1, kw
    assert L.sitk_block_mask(None, 16, 1, 10, 100, 4, 2, 64, 3, None) == -1
    assert L.sitk_block_mask_words(1, 10, 100, 3, 2, 64) == 0 and L.sitk_block_mask_words(2, 10, 6400, 4, 2, 64) == 2 * 2 * 2 * 100

    def desc(**kw):
        d = dict(B=1, Nq=10, Nk=100, H=4, Hk=2, block=64, scale=0.125, q=16, k=16, v=16, qs=rows, ks=rows, vs=rows, o=16, lse=16, mask=16,
                 pool=16)
        d.update(kw)
        return byref(rt.BlockAttn(*(d[n] for n, _ in rt.BlockAttn._fields_)))

    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(v=8), dict(o=None),
               dict(lse=None), dict(mask=None), dict(pool=None), dict(H=5), dict(qs=rt.BlockRows(0, 4, 64))):
        assert L.sitk_block_attention_fwd(desc(**kw), 16, 1 << 30, 1, None) == -1, kw
        assert L.sitk_block_attention_bwd(desc(**kw), 16, byref(rows), 16, 16, 16, 16, 1 << 30, 1, None) == -1, kw
    need = L.sitk_block_attention_bwd_ws_bytes(1, 10, 100, 4, 2, 64)
    assert L.sitk_block_attention_bwd(desc(), 16, byref(rows), 16, 16, 16, 16, need - 1, 1, None) == -1
    assert L.sitk_block_attention_bwd(desc(), 16, byref(rows), 16, None, 16, 16, need, 1, None) == -1
    assert L.sitk_block_attention_bwd(desc(), 8, byref(rows), 16, 16, 16, 16, need, 1, None) == -1


def test_act8_wgrad_without_rows(sitk_mods):
    """No rows, null operands as empty tensors have them: added to what is there nothing is launched, else only the join that writes the
    zeros (its launch fails here by name, where no device is)."""
    _, rt = sitk_mods
    for dtype in (0, 1, 2):
        for N in (24, 21):                                      # rows of whole 16-byte chunks and others
            assert rt.lib.sitk_act8_wgrad(None, N, None, None, 16, 40, 16, 0, N, 40, 1, None, 0, dtype, None) == 0, (dtype, N)
            if not torch.cuda.is_available():
                assert rt.lib.sitk_act8_wgrad(None, N, None, None, 16, 40, 16, 0, N, 40, 0, None, 0, dtype, None) == -2
                assert b"join" in rt.lib.sitk_last_error()


def test_unaligned_pools_codes_and_workspaces_are_refused(sitk_mods):
    """What include/sitk.h asks for: 16 bytes."""
    _, rt = sitk_mods
    L, rows = rt.lib, rt.BlockRows(0, 64, 64)
    assert L.sitk_act8_pack(16, 32, 24, 16, 3, 32, 1, None) == -1 and b"aligned" in L.sitk_last_error()
    assert L.sitk_act8_unpack(24, 16, 16, 32, 3, 32, 1, None) == -1
    assert L.sitk_act8_gelu_fwd(16, 32, 16, 32, 24, 16, 3, 32, 1, None) == -1
    assert L.sitk_act8_gelu_bwd(16, 32, 24, 16, 16, 32, 3, 32, 1, None) == -1
    assert L.sitk_block_select(16, C.byref(rows), 24, 16, 16, 1, 10, 100, 4, 2, 64, 3, 1, None) == -1 and b"aligned" in L.sitk_last_error()
    for pool, ws in ((24, 16), (16, 24)):
        d = rt.BlockAttn(1, 10, 1000, 4, 2, 64, 0.125, 16, 16, 16, rows, rows, rows, 16, 16, 16, pool)
        assert L.sitk_block_attention_fwd_ws_bytes(1, 10, 1000, 4, 2, 64, 1) > 0
        assert L.sitk_block_attention_fwd(C.byref(d), ws, 1 << 30, 1, None) == -1, (pool, ws)
        assert L.sitk_block_attention_bwd(C.byref(d), 16, C.byref(rows), 16, 16, 16, ws, 1 << 30, 1, None) == -1, (pool, ws)


def test_rope_inplace_overlaps(sitk_mods):
    """q and k that share memory are refused whatever they are slices of, a tensor that meets itself too; disjoint slices are not."""
    ops, rt = sitk_mods
    pos, f = torch.zeros(5, 2), ops.rope_freqs((4, 4), device="cpu")

    def call(q, k):
        return lambda: ops.rope_axes(q, k, pos, f, (4, 4), inplace=True)

    tok, smp, major = torch.zeros(2, 6, 3, 16), torch.zeros(3, 5, 3, 16), torch.zeros(2, 3, 6, 16).transpose(1, 2)
    wide = torch.zeros(2, 5, 64)
    q3 = wide[..., :48].view(2, 5, 3, 16)
    for q, k in ((tok[:, :5], tok[:, 1:]), (tok[:, 1:], tok[:, :5]), (smp[:2], smp[1:]), (major[:, :5], major[:, 1:]),   # a token, a sample apart
                 (q3, wide[..., 40:56].unsqueeze(2)), (q3, wide[..., 40:56].view(2, 5, 1, 16))):
        refused(rt, call(q, k), "share features")
    for q in (torch.zeros(1000).as_strided((2, 5, 3, 16), (240, 48, 8, 1)), torch.zeros(1000).as_strided((2, 5, 3, 16), (144, 48, 16, 1)),
              torch.zeros(1000).as_strided((2, 5, 2, 16), (8, 80, 16, 1))):
        refused(rt, call(q, None), "rows overlap")
    # the next token's first head is what a second head of k behind q's last one reaches
    far = torch.zeros(700)
    refused(rt, call(far.as_strided((2, 5, 3, 16), (320, 64, 16, 1)), far.as_strided((2, 5, 2, 16), (320, 64, 16, 1), 48)), "share features")
    packed = torch.zeros(2, 5, 8, 16)
    apart = [(packed[:, :, :4], packed[:, :, 4:6]), (packed[:, :, 4:6], packed[:, :, :4]), (packed[:, :, ::2], packed[:, :, 1::2]),
             (torch.zeros(2, 5, 3, 16), torch.zeros(2, 5, 1, 16)), (packed.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :4], packed[:, :, :1]),
             (packed[:1], packed[1:]), (wide[..., :48].view(2, 5, 3, 16), wide[..., 48:].unsqueeze(2))]
    twice = torch.zeros(2, 10, 3, 16)
    apart += [(twice[:, 0::2], twice[:, 1::2]), (twice[:, :5], twice[:, 5:]), (packed[:, :, :4], None)]
    for q, k in apart:
        refused(rt, call(q, k), "must live on a ROCm/HIP device")
    empty = torch.zeros(0, 5, 3, 16)
    refused(rt, call(empty, empty), "must live on a ROCm/HIP device")


def test_overlap_search_against_listing_every_byte(sitk_mods):
    """Random strided boxes in a small buffer: the answer of the search is that of the sets of addresses."""
    import random
    ops, _ = sitk_mods
    rng, buf, seen = random.Random(3), torch.zeros(400, dtype=torch.uint8), set()

    def box():
        while True:
            shape = [rng.randint(1, 3) for _ in range(3)] + [rng.randint(1, 4)]
            stride = [rng.choice([4, 5, 8, 12, 16, 24, 36, 48, 60]) for _ in range(3)] + [1]
            last = sum((n - 1) * t for n, t in zip(shape, stride))
            if last < 380:
                return buf.as_strided(shape, stride, rng.randint(0, 399 - last))

    def places(x):
        at = torch.tensor(x.storage_offset())
        for n, t in zip(x.shape, x.stride()):
            at = at[..., None] + torch.arange(n) * t
        return at.flatten().tolist()

    for _ in range(3000):
        a, b = box(), box()
        pa, pb = places(a), places(b)
        assert ops._share_features(a, b) == bool(set(pa) & set(pb)), (a.shape, a.stride(), b.shape, b.stride())
        assert ops._meets_itself(a) == (len(set(pa)) < len(pa)), (a.shape, a.stride())
        seen |= {(bool(set(pa) & set(pb)), len(set(pa)) < len(pa))}
    assert len(seen) == 4


def test_heads_as_the_kernels_read_them(sitk_mods):
    """Any layout of q, k, v comes out with features side by side, base and strides of whole 16 bytes, and the same values; aligned ones as
    they are."""
    ops, _ = sitk_mods
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for shape in ((1, 1, 1, 64), (2, 1, 1, 64), (1, 5, 1, 64), (1, 1, 3, 64), (2, 5, 3, 64)):
            x = torch.randn(shape).to(dtype)
            odd = torch.cat([x[..., :3], x], -1)[..., 3:]
            for y in (x, odd, x.transpose(1, 2).contiguous().transpose(1, 2), x.transpose(2, 3).contiguous().transpose(2, 3),
                      torch.cat([x, x[..., :1]], -1)[..., :64], x.flatten()[None, None, None, :64].expand(shape), odd[:, :1], odd[:1, :, :1]):
                z = ops._heads64(y, "x")
                m = 16 // z.element_size()
                assert torch.equal(z, y) and z.stride(3) == 1 and z.data_ptr() % 16 == 0 and all(s % m == 0 for s in z.stride()[:3])
            assert ops._heads64(x, "x") is x or any(s % 4 for s in x.stride()[:3])


def test_scales_that_leave_32_bits_are_refused(sitk_mods):
    ops, rt = sitk_mods
    k, q, rows = torch.zeros(2, 300, 2, 64), torch.zeros(2, 10, 4, 64), rt.BlockRows(0, 64, 64)
    pool = ops.BlockPool(torch.zeros(1 << 16, dtype=torch.uint8), 2, 300, 2, 64, torch.float32)
    sel = ops.BlockSelection(torch.zeros(2, 4, 10, 3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), pool)
    for scale in (1e-38, 1e-31, 2e30, 1e38):
        refused(rt, lambda: ops.block_attention_fwd(q, k, k, sel, scale), "scale")
        refused(rt, lambda: ops.block_attention_bwd(q, k, k, q, q, torch.zeros(2, 4, 10), sel, scale), "scale")
        d = rt.BlockAttn(1, 10, 100, 4, 2, 64, scale, 16, 16, 16, rows, rows, rows, 16, 16, 16, 16)
        assert rt.lib.sitk_block_attention_fwd(C.byref(d), 16, 1 << 30, 1, None) == -1 and b"scale" in rt.lib.sitk_last_error()
        assert rt.lib.sitk_block_attention_bwd(C.byref(d), 16, C.byref(rows), 16, 16, 16, 16, 1 << 30, 1, None) == -1
    for scale in (2.0 ** -100, 2.0 ** 100):
        refused(rt, lambda: ops.block_attention_fwd(q, k, k, sel, scale), "must live on")
