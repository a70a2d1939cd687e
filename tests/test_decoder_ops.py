"""Operators of one step of a served token model (seldon_core_amd.ops) against
plain 64-bit references, at the sizes, strides and indices where they can go
wrong.

Tolerances count roundings: u(type) = finfo.eps / 2 for the one rounding to the
output's type, and what the fp32 arithmetic before it can add, derived at each
test."""
import math

import pytest
import torch

from seldon_core_amd import ops

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


def u(dtype):
    return torch.finfo(dtype).eps / 2


def gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


def close(got, ref, dtype, atol):
    """|got - ref| <= u |ref| + atol everywhere; atol may be a tensor."""
    got, ref = got.double().cpu(), ref.double().cpu()
    over = (got - ref).abs() - (u(dtype) * ref.abs() + atol)
    assert torch.isfinite(got).all()
    assert float(over.max()) <= 0, f"over the tolerance by {float(over.max()):.3e}"


# ------------------------------------------------------- norm and rotation
def rope_inputs(g, T, hq, hk, D, rotary, dtype, fused=True):
    x = randn(g, T, (hq + 2 * hk) * D, dtype=dtype) * 3
    q, k = x[:, :hq * D].view(T, hq, D), x[:, hq * D:(hq + hk) * D].view(T, hk, D)
    w = [(1 + 0.3 * randn(g, D)).to(dtype) for _ in range(2)]
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    return x, q, k, w, inv


def rope_check(got, ref, dtype):
    # fp32 before the rounding: <= 40 additions of squares (half of their relative error after the root), rsqrt 2 ulp,
    # three products, the angle to 2^-22: under 40 * 2^-24 of the pair's magnitude, which the head's largest value bounds / sqrt(2)
    for a, b in zip(got, ref):
        close(a, b, dtype, 2.0 ** -18 * b.abs().amax(-1, keepdim=True).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hk,D,rotary", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 3, 1, 64, 32), (5, 4, 2, 80, 40),
                                              (33, 5, 5, 100, 50), (3, 2, 1, 72, 72), (9, 7, 1, 512, 512), (4, 2, 2, 510, 510),
                                              (2, 3, 3, 6, 2), (5, 2, 1, 96, 0), (4100, 3, 2, 64, 64), (1025, 2, 1, 258, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
def test_qk_norm_rope(T, hq, hk, D, rotary, interleaved, dtype):
    g = gen(T, hq, hk, D, rotary)
    dt = DT[dtype]
    x, q, k, w, inv = rope_inputs(g, T, hq, hk, D, rotary, dt)
    pos = torch.randint(0, 1_000_000, (T,), generator=g)
    xd = x.cuda()
    qd, kd = xd[:, :hq * D].view(T, hq, D), xd[:, hq * D:(hq + hk) * D].view(T, hk, D)
    got = ops.qk_norm_rope(qd, kd, w[0].cuda(), w[1].cuda(), pos.cuda(), inv.cuda(), interleaved=interleaved)
    assert got[0].dtype == dt and got[0].is_contiguous() and got[1].shape == k.shape
    rope_check(got, ops.token_step.qk_norm_rope_ref(q, k, w[0], w[1], pos, inv, interleaved=interleaved), dt)
    assert torch.equal(xd.cpu(), x)  # the inputs stay


@pytest.mark.gpu
def test_qk_norm_rope_in_place_weights_and_index_types():
    g = gen(11)
    T, hq, hk, D = 19, 6, 2, 128
    x, q, k, w, inv = rope_inputs(g, T, hq, hk, D, 64, torch.bfloat16)
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
    ref = ops.token_step.qk_norm_rope_ref(q, k, None, None, pos, inv.float())
    xd = x.cuda()
    qd, kd = xd[:, :hq * D].view(T, hq, D), xd[:, hq * D:(hq + hk) * D].view(T, hk, D)
    got = ops.qk_norm_rope(qd, kd, None, None, pos.cuda(), inv.float().cuda(), out=(qd, kd))
    assert got[0].data_ptr() == xd.data_ptr()
    rope_check(got, ref, torch.bfloat16)
    assert torch.equal(xd[:, (hq + hk) * D:].cpu(), x[:, (hq + hk) * D:])  # the values beside them stay
    # heads in front of tokens, fp32 weights for one of the two
    qt = q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    kt = k.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    wf = w[0].float()
    got = ops.qk_norm_rope(qt, kt, wf.cuda(), None, pos.cuda(), inv.cuda())
    rope_check(got, ops.token_step.qk_norm_rope_ref(q, k, wf, None, pos, inv), torch.bfloat16)
    # an odd storage offset: no vector is aligned
    flat = torch.zeros(T * hq * D + 1, dtype=torch.bfloat16).cuda()
    qo = flat[1:].view(T, hq, D)
    qo.copy_(q)
    got = ops.qk_norm_rope(qo, kt, None, None, pos.cuda(), inv.float().cuda())
    rope_check(got, ref, torch.bfloat16)


@pytest.mark.gpu
def test_qk_norm_rope_far_positions_zero_rows_and_nothing():
    g = gen(12)
    x, q, k, w, inv = rope_inputs(g, 4, 2, 1, 64, 64, torch.float32)
    q = q.clone()
    q[1] = 0  # a head of zeros stays zeros
    pos = torch.tensor([0, 1, 2 ** 31 - 1, -7])
    got = ops.qk_norm_rope(q.cuda(), k.cuda(), None, None, pos.cuda(), inv.cuda())
    # at 2^31 the product with inv_freq is a 53-bit number of 2^29 radians: an error of 2^-24 more
    rope_check(got, ops.token_step.qk_norm_rope_ref(q, k, None, None, pos, inv), torch.float32)
    assert not got[0][1].any()
    e = torch.empty((0, 2, 64), device="cuda")
    a, b = ops.qk_norm_rope(e, e, None, None, torch.empty(0, dtype=torch.int64, device="cuda"), inv.cuda())
    assert a.shape == b.shape == (0, 2, 64)


# ------------------------------------------------------------------- cache
def values(codes, scales):
    return codes.double() * scales.double()[..., None]


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=1e300), torch.nan_to_num(b.double(), nan=1e300))


@pytest.mark.gpu
@pytest.mark.parametrize("T,pages,page,heads,dim", [(1, 1, 1, 1, 1), (5, 3, 16, 2, 64), (64, 40, 24, 8, 128), (33, 64, 1, 3, 80),
                                                    (7, 4, 5, 1, 33), (300, 30, 16, 4, 256), (6, 2, 7, 2, 512), (9, 3, 8, 3, 511)])
@pytest.mark.parametrize("cache", ["fp32", "fp16", "bf16", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", list(DT))
def test_kv_cache_write_and_read(T, pages, page, heads, dim, cache, dtype):
    g = gen(T, pages, page, heads, dim)
    dt, ct = DT[dtype], {**DT, "e4m3": E4M3, "int8": torch.int8}[cache]
    c = ops.kv_cache(pages, page, heads, dim, dtype=ct)
    k, v = randn(g, T, heads, dim, dtype=dt), randn(g, T, heads, dim, dtype=dt) * 37
    k[:, :1] = 0  # heads of zeros
    slots = torch.randperm(pages * page, generator=g)[:T]
    assert len(slots) == T
    slots[T // 2] = -1  # padding
    assert ops.kv_cache_write(c, k.cuda(), v.cuda(), slots.cuda()) is c
    kept = slots >= 0
    for x, codes, scales in ((k, c.k, c.k_scales), (v, c.v, c.v_scales)):
        flat = codes.cpu().view(-1, heads, dim)
        if scales is None:
            want = torch.zeros((pages * page, heads, dim), dtype=ct)
            want[slots[kept]] = x[kept].to(ct)
            assert torch.equal(flat, want)
        else:
            qc, qs = ops.token_step.kv_quantise_ref(x[kept], ct)
            want = torch.zeros((pages * page, heads, dim))
            ws = torch.ones((pages * page, heads))
            want[slots[kept]], ws[slots[kept]] = qc.float(), qs
            assert torch.equal(flat.float(), want) and torch.equal(scales.cpu().view(-1, heads), ws)
            # e4m3: half a step of the value, 2^-4 of it, or where it is subnormal 2^-10 scales, with scale <= top / 224.
            # int8: |code - x / s| <= 1/2 + 127 * 2^-24 (the quotient's own rounding) < 1/2 (1 + 2^-16) and
            # s <= top / 127 (1 + 2^-24)^2, so |code * s - x| <= top / 254 (1 + 2^-15).
            got = values(flat, scales.cpu().view(-1, heads))[slots[kept]]
            top = x[kept].double().abs().amax(-1, keepdim=True)
            step = x[kept].double().abs() * 2.0 ** -4 + top * 2.0 ** -17 if ct == E4M3 else top / 254 * (1 + 2.0 ** -15)
            assert bool((got - x[kept].double()).abs().le(step).all())
    # what comes back, with slots outside of the cache in between and an order of its own
    ask = torch.cat((slots.flip(0), torch.tensor([pages * page, -5, 2 ** 40])))
    for out in (dt, None):
        kr, vr = ops.kv_cache_read(c, ask.cuda(), dtype=out)
        od = out or (ct if ct.itemsize > 1 else torch.bfloat16)
        assert kr.dtype == od
        for r, codes, scales in ((kr, c.k, c.k_scales), (vr, c.v, c.v_scales)):
            flat = codes.cpu().view(-1, heads, dim).float()
            if scales is not None:
                flat = flat * scales.cpu().view(-1, heads)[..., None]
            ok = (ask >= 0) & (ask < pages * page)
            want = torch.where(ok[:, None, None], flat[torch.where(ok, ask, 0)], torch.zeros(())).to(od)
            assert torch.equal(r.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["e4m3", "int8"])
def test_kv_cache_scales_over_the_whole_range(cache):
    """Every magnitude that bf16 has, borders of the scale's steps, and values that are not finite."""
    ct = {"e4m3": E4M3, "int8": torch.int8}[cache]
    tops = [0.0, 1e-40, 2.0 ** -126, 2.0 ** -120, 1e-30, 1.0, 448.0, 449.0, 450.0, 447.9, 1.75, 1.7578125, 1e30, 2.0 ** 126, 3e38]
    bad = [math.inf, -math.inf, math.nan]
    k = torch.zeros((len(tops) + len(bad), 1, 32))
    for i, t in enumerate(tops + bad):
        k[i, 0] = torch.linspace(-1, 1, 32) * (t if math.isfinite(t) else 1.0)
        k[i, 0, 5] = t
    c = ops.kv_cache(2, 16, 1, 32, dtype=ct)
    slots = torch.arange(len(k), dtype=torch.int32)
    ops.kv_cache_write(c, k.cuda(), k.cuda(), slots.cuda())
    codes, scales = ops.token_step.kv_quantise_ref(k, ct)
    n = len(k)
    assert same(c.k_scales.cpu().view(-1, 1)[:n], scales) and same(c.v.cpu().view(-1, 1, 32)[:n].float(), codes.float())
    kr, _ = ops.kv_cache_read(c, slots.cuda(), dtype=torch.float32)
    assert torch.isfinite(kr[:len(tops) - 1]).all() and kr[len(tops):].isnan().all()


@pytest.mark.gpu
def test_kv_cache_layouts_and_far_offsets():
    """Pages of a head together, rows out of a fused projection, and a pool past 2^31 elements."""
    g = gen(5)
    T, heads, dim, pages, page = 40, 4, 64, 6, 16
    base = [torch.zeros((pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    sc = [torch.ones((pages, heads, page), device="cuda") for _ in range(2)]
    c = ops.KVCache(*(b.transpose(1, 2) for b in base), *(s.transpose(1, 2) for s in sc))
    x = randn(g, T, 3 * heads * dim, dtype=torch.bfloat16).cuda()
    k, v = x[:, heads * dim:2 * heads * dim].view(T, heads, dim), x[:, 2 * heads * dim:].view(T, heads, dim)
    slots = torch.randperm(pages * page, generator=g)[:T].cuda()
    ops.kv_cache_write(c, k, v, slots)
    codes, scales = ops.token_step.kv_quantise_ref(v.cpu(), torch.int8)
    s = slots.cpu()
    assert torch.equal(base[1].cpu()[s // page, :, s % page], codes)
    assert torch.equal(sc[1].cpu()[s // page, :, s % page], scales)
    kr, vr = ops.kv_cache_read(c, slots)
    assert torch.equal(vr.cpu(), (codes.float() * scales[..., None]).bfloat16())

    pages, page, heads, dim = 1200, 1024, 8, 256  # 2.5 G elements each for k and v
    c = ops.KVCache(*(torch.empty((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    slots = torch.tensor([0, pages * page - 1, pages * page // 2, 1_100_000], device="cuda")
    k, v = (randn(g, 4, heads, dim, dtype=torch.bfloat16).cuda() for _ in range(2))
    ops.kv_cache_write(c, k, v, slots)
    assert torch.equal(c.k[-1, -1], k[1]) and torch.equal(c.v[1_100_000 // page, 1_100_000 % page], v[3])
    kr, vr = ops.kv_cache_read(c, slots)
    assert torch.equal(kr, k) and torch.equal(vr, v)
