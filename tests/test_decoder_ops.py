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
    """|got - ref| <= u |ref| + atol everywhere (atol may be a tensor), and NaN exactly where the reference has it."""
    got, ref = got.double().cpu(), ref.double().cpu()
    over = (got - ref).abs() - (u(dtype) * ref.abs() + atol)
    assert torch.equal(got.isnan(), ref.isnan()) and not got.isinf().any()
    over = over[~ref.isnan()]
    assert not len(over) or float(over.max()) <= 0, f"over the tolerance by {float(over.max()):.3e}"


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
        flat = codes.cpu().reshape(-1, heads, dim)
        if scales is None:
            want = torch.zeros((pages * page, heads, dim), dtype=ct)
            want[slots[kept]] = x[kept].to(ct)
            assert torch.equal(flat, want)
        else:
            qc, qs = ops.token_step.kv_quantise_ref(x[kept], ct)
            want = torch.zeros((pages * page, heads, dim))
            ws = torch.ones((pages * page, heads))
            want[slots[kept]], ws[slots[kept]] = qc.float(), qs
            assert torch.equal(flat.float(), want) and torch.equal(scales.cpu().reshape(-1, heads), ws)
            # e4m3: half a step of the value, 2^-4 of it, or where it is subnormal 2^-10 scales, with scale <= top / 224.
            # int8: |code - x / s| <= 1/2 + 127 * 2^-24 (the quotient's own rounding) < 1/2 (1 + 2^-16) and
            # s <= top / 127 (1 + 2^-24)^2, so |code * s - x| <= top / 254 (1 + 2^-15).
            got = values(flat, scales.cpu().reshape(-1, heads))[slots[kept]]
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
            flat = codes.cpu().reshape(-1, heads, dim).float()
            if scales is not None:
                flat = flat * scales.cpu().reshape(-1, heads)[..., None]
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
    assert same(c.k_scales.cpu().reshape(-1, 1)[:n], scales) and same(c.v.cpu().reshape(-1, 1, 32)[:n].float(), codes.float())
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


# --------------------------------------------------------------- attention
def attention_inputs(g, lens, Hq, H, D, page, dtype, cache, spare=3, sharp=2.0, heads_first=False):
    """A pool with NaN wherever no request has a token, and a table with -1 behind each request's pages."""
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + spare
    W = max(1, max(need))
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    at = 0
    used = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[at:at + need[b]].int()
        at += need[b]
        t = torch.arange(max(n, 0))
        used[table[b, t // page].long(), t % page] = True
    kv = []
    for _ in range(2):
        x = randn(g, pages, page, H, D, dtype=dtype)
        if cache == "same":
            x[~used] = math.nan
            kv.append((x, None))
        else:
            codes, scales = ops.token_step.kv_quantise_ref(x, E4M3 if cache == "e4m3" else torch.int8)
            scales[~used] = math.nan
            if cache == "e4m3":
                codes.view(torch.uint8)[~used] = 0x7f  # NaN
            kv.append((codes, scales))
    q = (randn(g, len(lens), Hq, D) * sharp).to(dtype)
    c = ops.KVCache(kv[0][0], kv[1][0], kv[0][1], kv[1][1])
    return q, c, table, torch.tensor(lens, dtype=torch.int32)


def to_gpu(c, heads_first=False):
    if heads_first:  # the pages of a head together
        return ops.KVCache(*(None if x is None else x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in c))
    return ops.KVCache(*(None if x is None else x.cuda() for x in c))


def attention_check(got, lse, q, c, table, lens, scale=None, window=0):
    ref, rlse, mag = ops.token_step.paged_attention_ref(q, c, table, lens, scale, window)
    D = q.shape[-1]
    n = min(int(lens.clamp_min(0).max()), table.shape[1] * c.k.shape[1]) + 1
    sc = D ** -0.5 if scale is None else abs(scale)
    k = c.k.double() if c.k_scales is None else c.k.float().double() * c.k_scales.double()[..., None]
    # |s| and the sum of |q||k| by Cauchy and Schwarz; an fp32 sum of D products is off by at most (D + 3) 2^-24 of that, and
    # as much again enters through the softmax's total.  The sum over n tokens adds n 2^-24, exp2 and the joins under 64 * 2^-24,
    # the split weights 2^-16.  All of it relative to the sum of |weight * value|.
    s = sc * float(q.double().norm(dim=-1).max()) * float(torch.nan_to_num(k, posinf=0.0, neginf=0.0).norm(dim=-1).max())
    rel = (2 * (D + 3) * s + n + 64) * 2.0 ** -24 + 2.0 ** -16
    close(got, ref, q.dtype, rel * mag)
    if lse is not None:
        lse = lse.cpu().double()
        seen = torch.isfinite(rlse)
        assert torch.equal(lse.isnan(), rlse.isnan()) and torch.equal(lse == -math.inf, rlse == -math.inf)
        assert bool(((lse - rlse)[seen].abs() <= ((D + 3) * s + n + 64) * 2.0 ** -24 + rlse[seen].abs() * 2.0 ** -22).all())
    return ref


ATTENTION = [  # lengths, query heads, key heads, dim, page, window
    ([1], 1, 1, 64, 16, 0), ([0], 4, 2, 128, 16, 0), ([5, 0, 1], 8, 2, 128, 16, 0), ([128, 127, 129, 31, 32, 33], 4, 4, 64, 24, 0),
    ([1000, 3, 256, 0, 511], 32, 8, 128, 16, 0), ([700], 7, 1, 128, 64, 0), ([300, 40], 40, 2, 64, 1, 0),
    ([4097], 16, 1, 256, 32, 0), ([90, 2000], 6, 2, 80, 7, 0), ([1500, 10, 0], 12, 12, 96, 48, 100),
    ([600, 601, 5], 4, 2, 256, 16, 1), ([2500], 8, 8, 64, 16, 777), ([64] * 37, 8, 4, 128, 16, 0),
    ([3, 700] * 150, 2, 1, 64, 8, 0), ([140] * 5, 34, 1, 48, 16, 129), ([333], 5, 1, 16, 16, 0), ([50], 3, 3, 208, 5, 60)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
@pytest.mark.parametrize("cache", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_paged_attention(case, cache, dtype):
    lens, Hq, H, D, page, window = case
    g = gen(len(lens), *case[1:])
    q, c, table, lengths = attention_inputs(g, lens, Hq, H, D, page, DT[dtype], cache)
    got, lse = ops.paged_attention(q.cuda(), to_gpu(c, heads_first=page % 2 == 0), table.cuda(), lengths.cuda(), window=window,
                                   return_lse=True)
    attention_check(got, lse, q, c, table, lengths, window=window)
    assert not got[lengths.cuda() == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "int8"])
def test_paged_attention_bad_pages_lengths_and_strides(cache):
    g = gen(3, 1)
    lens = [200, 70, 33, 129, 64]
    q, c, table, lengths = attention_inputs(g, lens, 8, 2, 128, 16, torch.bfloat16, cache)
    pages = c.k.shape[0]
    table[0, 3], table[0, 7], table[1, 0] = pages, -2, 2 ** 31 - 1  # pages that do not exist: their tokens are left out
    table[2] = -1  # nothing is left of this one
    lengths[3] = 10 ** 9  # longer than the table: its end, whose last real page holds NaN behind token 129: so does the output
    lengths[4] = -5  # nothing
    wide = torch.full((5, table.shape[1] + 3), 10 ** 6, dtype=torch.int32)
    wide[:, :-3] = table
    qs = torch.full((5, 8, 3 * 128), math.nan, dtype=torch.bfloat16)
    qs[:, :, 128:256] = q
    out = torch.full((5, 8, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    got, lse = ops.paged_attention(qs.cuda()[:, :, 128:256], to_gpu(c), wide.cuda()[:, :-3], lengths.cuda(), scale=0.25,
                                   return_lse=True, out=out)
    assert got is out
    attention_check(got, lse, q, c, table, lengths, scale=0.25)
    assert got[3].isnan().all() and not got[0].isnan().any()
    assert not got[2].any() and not got[4].any()
    # queries that start at an odd element
    qo = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    qo.copy_(q)
    again = ops.paged_attention(qo, to_gpu(c), table.cuda(), lengths.cuda(), scale=0.25)
    assert torch.equal(again.nan_to_num(7.0), got.nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_paged_attention_scores_far_apart(dtype):
    """One token far above a long flat tail, rising and falling scores, and scores of thousands."""
    g = gen(8)
    n, D = 5000, 64
    dt = DT[dtype]
    for kind in ("peak first", "peak last", "rising", "falling", "huge"):
        q, c, table, lengths = attention_inputs(g, [n], 2, 1, D, 16, dt, "same", sharp=0.0)
        q[..., 0] = 8
        slots = table[0, torch.arange(n) // 16].long() * 16 + torch.arange(n) % 16
        k = c.k.view(-1, D)
        k[slots] = 0
        s = torch.zeros(n)
        if kind == "peak first":
            s[3] = 17
        elif kind == "peak last":
            s[n - 2] = 17
        elif kind == "huge":
            s = torch.randn(n, generator=g) * 3000
        else:
            s = torch.linspace(-40, 40, n) * (1 if kind == "rising" else -1)
        k[slots, 0] = s.to(dt)
        got, lse = ops.paged_attention(q.cuda(), to_gpu(c), table.cuda(), lengths.cuda(), return_lse=True)
        attention_check(got, lse, q, c, table, lengths)


@pytest.mark.gpu
def test_paged_attention_pool_past_2_31_elements():
    g = gen(9)
    pages, page, H, D = 70000, 32, 8, 128  # 2.3 G elements
    c = ops.KVCache(*(torch.zeros((pages, page, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    n = 300
    table = torch.tensor([[pages - 1 - 7 * i for i in range(10)]], dtype=torch.int32)
    t = torch.arange(n)
    slots = table[0, t // page].long() * page + t % page
    k, v = (randn(g, n, H, D, dtype=torch.bfloat16) for _ in range(2))
    ops.kv_cache_write(c, k.cuda(), v.cuda(), slots.cuda())
    q = randn(g, 1, 16, D, dtype=torch.bfloat16)
    got = ops.paged_attention(q.cuda(), c, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    small = ops.KVCache(*(torch.zeros((10, page, H, D), dtype=torch.bfloat16) for _ in range(2)))
    small.k.view(-1, H, D)[:n], small.v.view(-1, H, D)[:n] = k, v
    attention_check(got, None, q, small, torch.arange(10, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32))


# ---------------------------------------------------------------- adapters
LORA = [  # rows, inner, outer, rank, adapters, mixed
    (1, 1, 1, 1, 1, True), (1, 4096, 4096, 16, 4, True), (64, 1024, 640, 16, 32, True), (17, 200, 77, 12, 3, True),
    (333, 1001, 503, 9, 5, False), (16, 512, 512, 64, 16, True), (40, 300, 1030, 100, 2, False), (5, 4104, 72, 128, 5, True),
    (1025, 512, 384, 8, 3, False), (1100, 320, 200, 32, 40, True), (2000, 264, 1100, 64, 7, False), (1030, 130, 66, 128, 2, True),
    (1024, 64, 64, 33, 1000, True), (3, 8200, 64, 5, 2, True),
    (4099, 72, 80, 8, 300, True), (1025, 32, 16, 4, 2000, True), (1026, 40, 24, 4, 2001, True), (1100, 33, 17, 4, 1, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LORA, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", list(DT))
def test_lora_add(case, dtype):
    T, K, M, r, N, mixed = case
    dt = DT[dtype]
    g = gen(*case[:5])
    x, y = randn(g, T, K, dtype=dt), randn(g, T, M, dtype=dt)
    A, B = (randn(g, N, r, K) * K ** -0.5).to(dt), (randn(g, N, M, r) * r ** -0.5).to(dt)
    ids = torch.randint(-1, N + 1, (T,), generator=g) if mixed else torch.arange(T) * N // T
    if T > 3:
        ids[T // 3] = -7
    scales = randn(g, N)
    want, mag = ops.token_step.lora_add_ref(y, x, A, B, ids, scales)
    yd = y.cuda()
    got = ops.lora_add(yd, x.cuda(), A.cuda(), B.cuda(), ids.cuda(), scales.cuda())
    assert torch.equal(yd.cpu(), y)
    # the two sums in fp32 ((K + r + 8) 2^-24 of the sum of magnitudes), h in two 16-bit parts: 2^-16 of it (bf16), or 2^-24 of the
    # row's largest h for fp16, whose remainder may be subnormal
    atol = (K + r + 8) * 2.0 ** -24 * mag + (2.0 ** -16 * mag if dt == torch.bfloat16 else 0)
    if dt == torch.float16:
        ok = (ids >= 0) & (ids < N)
        i = torch.where(ok, ids, 0)
        for t in range(T):
            if ok[t]:
                h = (A[i[t]].double() @ x[t].double()).abs().max() * abs(scales[i[t]].double())
                atol[t] += 2.0 ** -23 * h * B[i[t]].double().abs().sum(-1)
    close(got, want, dt, atol + 2.0 ** -24 * want.abs())
    untouched = (ids < 0) | (ids >= N)
    assert torch.equal(got.cpu()[untouched], y[untouched])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 512, 513, 1500])
def test_lora_add_strides_in_place_and_index_types(T):
    """A part of a fused projection changed in place, and its neighbours left as they were."""
    g = gen(T)
    K, M, r, N = 128, 192, 16, 4
    x, y = randn(g, T, K + 8, dtype=torch.bfloat16), randn(g, T, 3 * M, dtype=torch.bfloat16)
    A, B = randn(g, N, r, K, dtype=torch.bfloat16) * 0.1, randn(g, N, M, r, dtype=torch.bfloat16)
    ids = (torch.arange(T) % (N + 1) - 1).int()
    want, mag = ops.token_step.lora_add_ref(y[:, M:2 * M], x[:, 8:], A, B, ids)
    for off in (0, 1):  # aligned rows, and rows that no vector fits
        buf = torch.zeros(T * 3 * M + off, dtype=torch.bfloat16, device="cuda")
        yd = buf[off:].view(T, 3 * M)
        yd.copy_(y)
        part = yd[:, M:2 * M]
        got = ops.lora_add(part, x.cuda()[:, 8:], A.cuda(), B.cuda(), ids.cuda(), out=part)
        assert got.data_ptr() == part.data_ptr()
        close(part, want, torch.bfloat16, (2.0 ** -16 + (K + r + 8) * 2.0 ** -24) * mag + 2.0 ** -24 * want.abs())
        assert torch.equal(yd.cpu()[:, :M], y[:, :M]) and torch.equal(yd.cpu()[:, 2 * M:], y[:, 2 * M:])
        assert torch.equal(part.cpu()[ids < 0], y[:, M:2 * M][ids < 0])


@pytest.mark.gpu
def test_lora_add_large_and_infinite_values():
    """fp16: an h far beyond fp16's range that B brings back; infinities reach only their own rows and columns."""
    g = gen(77)
    T, K, M, r = 5, 256, 64, 8
    x = (randn(g, T, K).abs() * 100 + 100).half()
    A, B = torch.full((1, r, K), 30.0).half(), (randn(g, 1, M, r) * 1e-4).half()
    y, ids = randn(g, T, M).half(), torch.zeros(T, dtype=torch.int32)
    want, mag = ops.token_step.lora_add_ref(y, x, A, B, ids)  # h is about 10^6
    got = ops.lora_add(y.cuda(), x.cuda(), A.cuda(), B.cuda(), ids.cuda())
    close(got, want, torch.float16, ((K + r + 8) * 2.0 ** -24 + 2.0 ** -21) * mag + 2.0 ** -24 * want.abs())
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        xi = x.to(dt)
        xi[2, 3] = math.inf
        got = ops.lora_add(y.to(dt).cuda(), xi.cuda(), A.to(dt).cuda(), B.abs().clamp_min(1e-4).to(dt).cuda(), ids.cuda()).cpu()
        assert (got[2] == math.inf).all() and torch.isfinite(got[[0, 1, 3, 4]]).all()
    e = ops.lora_add(torch.empty((0, M), device="cuda"), torch.empty((0, K), device="cuda"), A.float().cuda(), B.float().cuda(),
                     torch.empty(0, dtype=torch.int32, device="cuda"))
    assert e.shape == (0, M)


# ----------------------------------------------------- together, as they are used
class Step(torch.nn.Module):
    """One decoder attention block over a cache that it keeps: projection with adapters, norm and rotation, cache, attention."""

    def __init__(self, hidden, Hq, H, D, tenants, pages, page, cache, g):
        super().__init__()
        self.Hq, self.H, self.D, self.page = Hq, H, D, page
        n = (Hq + 2 * H) * D
        self.w = (randn(g, n, hidden) * hidden ** -0.5).bfloat16().cuda()
        self.A, self.B = (randn(g, tenants, 8, hidden) * hidden ** -0.5).bfloat16().cuda(), (randn(g, tenants, n, 8) * 0.3).bfloat16().cuda()
        self.qn, self.kn = ((1 + 0.1 * randn(g, D)).bfloat16().cuda() for _ in range(2))
        self.inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).cuda()
        self.cache = ops.kv_cache(pages, page, H, D, dtype=cache)

    def forward(self, x, tenant, positions, table):
        if not torch.cuda.is_current_stream_capturing():  # inputs and cache are made on the default stream
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        Hq, H, D = self.Hq, self.H, self.D
        y = x @ self.w.T
        y = ops.lora_add(y, x, self.A, self.B, tenant, out=y).view(len(x), -1, D)
        q, k = ops.qk_norm_rope(y[:, :Hq], y[:, Hq:Hq + H], self.qn, self.kn, positions, self.inv)
        at = positions.clamp_min(0).long()  # padding has no place in the table
        slots = table.long().gather(1, at[:, None] // self.page)[:, 0] * self.page + at % self.page
        slots = torch.where(positions >= 0, slots, -1)
        ops.kv_cache_write(self.cache, k, y[:, Hq + H:], slots)
        return ops.paged_attention(q, self.cache, table, positions + 1)


def step_inputs(g, T, tenants, table_width, page, at):
    """Requests at position `at` + i, the last one padding."""
    x = randn(g, T, 256, dtype=torch.bfloat16).cuda()
    pos = (at + torch.arange(T) * 3).int()
    pos[-1] = -1
    return x, (torch.arange(T) % (tenants + 1) - 1).int().cuda(), pos.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [torch.bfloat16, E4M3, torch.int8])
def test_steps_together_and_replayed(cache):
    """Eight decode steps eagerly against 64 bits, then the same steps as replays of one captured graph: the same bits."""
    T, page, W, Hq, H, D, tenants = 5, 16, 4, 8, 2, 64, 3
    g = gen(21)
    m = Step(256, Hq, H, D, tenants, T * W, page, cache, g)
    table = torch.randperm(T * W, generator=g).int().view(T, W).cuda()
    inputs = [step_inputs(g, T, tenants, W, page, 7 + i) for i in range(8)]
    for i, (x, tenant, pos) in enumerate(inputs):  # the prompts' tokens: random rows at the positions before
        if i == 0:
            for t in range(T - 1):
                n = int(pos[t])
                s = table[t].long().cpu()[torch.arange(n) // page] * page + torch.arange(n) % page
                ops.kv_cache_write(m.cache, *(randn(g, n, H, D, dtype=torch.bfloat16).cuda() for _ in range(2)), s.cuda())
    start = [None if c is None else c.clone() for c in m.cache]
    outs = []
    with torch.no_grad():
        for x, tenant, pos in inputs:
            out = m(x, tenant, pos, table)
            outs.append(out.clone())
            # the last piece against 64 bits on the cache as it is
            y = x @ m.w.T
            ops.lora_add(y, x, m.A, m.B, tenant, out=y)
            q, _ = ops.qk_norm_rope(y.view(T, -1, D)[:, :Hq], y.view(T, -1, D)[:, Hq:Hq + H], m.qn, m.kn, pos, m.inv)
            c = ops.KVCache(*(None if t is None else t.cpu() for t in m.cache))
            attention_check(out, None, q.cpu(), c, table.cpu(), pos.cpu() + 1)
            assert not out[-1].any()
    end = [None if c is None else c.clone() for c in m.cache]
    # captured: static inputs, replayed with eager work in between
    sx, st, sp = (t.clone() for t in inputs[0])
    side = torch.cuda.Stream()
    with torch.no_grad(), torch.cuda.stream(side):
        m(sx, st, sp, table)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=side):
        sy = m(sx, st, sp, table)
    for c, b in zip(m.cache, start):
        if c is not None:
            c.copy_(b)
    for (x, tenant, pos), want in zip(inputs, outs):
        sx.copy_(x), st.copy_(tenant), sp.copy_(pos)
        graph.replay()
        junk = ops.lora_add(x @ m.w.T, x, m.A, m.B, tenant)  # eager work of the same shapes
        torch.cuda.synchronize()
        assert torch.equal(sy, want) and junk.shape[0] == T
    for c, b in zip(m.cache, end):
        assert c is None or torch.equal(c.float(), b.float())


@pytest.mark.gpu
def test_two_graphs_and_two_streams_share_nothing():
    """Two captured calls replayed at once on two streams give what each gives alone."""
    g = gen(33)
    cases = []
    for lens in ([3000, 17, 400], [1200, 2500, 1]):
        q, c, table, lengths = attention_inputs(g, lens, 16, 4, 128, 16, torch.bfloat16, "same")
        cases.append((q.cuda(), to_gpu(c), table.cuda(), lengths.cuda()))
    want = [ops.paged_attention(*c) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for c, s in zip(cases, streams):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(ops.paged_attention(*c))
        graphs.append(graph)
    for _ in range(5):
        for o in outs:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


@pytest.mark.gpu
def test_served_module_replays_adapters_through_graphs():
    """A torch module of linear layers with an adapter beside each, served by GraphedModule."""
    from seldon_core_amd.models.graphed import GraphedModule

    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a = torch.nn.Linear(64, 96)
            self.A, self.B = torch.nn.Parameter(torch.randn(2, 8, 64) * 0.1), torch.nn.Parameter(torch.randn(2, 96, 8))

        def forward(self, x):  # the last column says whose row it is
            y = self.a(x[:, :-1])
            return ops.lora_add(y, x[:, :-1], self.A, self.B, x[:, -1].to(torch.int32))

    m = GraphedModule(M(), max_batch=16)
    X = torch.randn(37, 65)
    X[:, -1] = torch.arange(37) % 3 - 1
    got = m(X.numpy())
    assert m.graph_error is None and m.replays >= 3
    mod = m.module.cpu()
    x, ids = X[:, :-1], X[:, -1].int()
    want, mag = ops.token_step.lora_add_ref((x.double() @ mod.a.weight.double().T + mod.a.bias.double()).detach(), x, mod.A.detach(),
                                            mod.B.detach(), ids)
    lin = x.abs().double() @ mod.a.weight.detach().abs().double().T + mod.a.bias.detach().abs().double()
    close(torch.from_numpy(got), want, torch.float32, 200 * 2.0 ** -24 * (mag + lin))  # sums of 64 and 8 products, and y's own


# ---------------------------------------------------------------- refusals
@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_refusals_before_anything_is_launched():
    """On fake GPU tensors: every refusal comes from the host's checks."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.qk_norm_rope(torch.zeros(2, 2, 4), torch.zeros(2, 2, 4), None, None, torch.zeros(2), torch.zeros(2))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.lora_add(*[torch.zeros(2, 2)] * 5)
    with FakeTensorMode():
        def t(*shape, dtype=bf):
            return torch.empty(shape, dtype=dtype, device="cuda")

        q, k, pos, inv = t(4, 8, 64), t(4, 2, 64), t(4, dtype=i32), t(32, dtype=f32)

        def refuse(error, match, fn, *a, **kw):
            with pytest.raises(error, match=match):
                fn(*a, **kw)

        rope = ops.qk_norm_rope
        refuse(TypeError, "k must be", rope, q, t(4, 2, 64, dtype=f32), None, None, pos, inv)
        refuse(TypeError, "q must be", rope, t(4, 8, 64, dtype=torch.float64), k, None, None, pos, inv)
        refuse(ValueError, "agree", rope, q, t(5, 2, 64), None, None, pos, inv)
        refuse(ValueError, "even", rope, t(4, 8, 63), t(4, 2, 63), None, None, pos, inv)
        refuse(ValueError, "even", rope, t(4, 8, 514), t(4, 2, 514), None, None, pos, inv)
        refuse(ValueError, "last dimension", rope, t(4, 64, 8).transpose(1, 2), k, None, None, pos, inv)
        refuse(ValueError, "q_weight must have", rope, q, k, t(63), None, pos, inv)
        refuse(TypeError, "one type", rope, q, k, t(64), t(64, dtype=f32), pos, inv)
        refuse(ValueError, "positions must have", rope, q, k, None, None, t(5, dtype=i32), inv)
        refuse(TypeError, "positions", rope, q, k, None, None, t(4, dtype=f32), inv)
        refuse(ValueError, "turns", rope, q, k, None, None, pos, t(33, dtype=f32))
        refuse(ValueError, r"out\[0\]", rope, q, k, None, None, pos, inv, out=(t(4, 8, 32), k))
        refuse(RuntimeError, "forward only", rope, q.clone().requires_grad_(), k, None, None, pos, inv)

        c, c8 = ops.KVCache(t(5, 16, 2, 64), t(5, 16, 2, 64)), ops.KVCache(
            *(t(5, 16, 2, 64, dtype=torch.int8) for _ in range(2)), *(t(5, 16, 2, dtype=f32) for _ in range(2)))
        write, read, v, slots = ops.kv_cache_write, ops.kv_cache_read, t(4, 2, 64), t(4, dtype=i32)
        refuse(ValueError, "no scales", write, ops.KVCache(c.k, c.v, c8.k_scales, c8.v_scales), k, v, slots)
        refuse(ValueError, "has scales", write, ops.KVCache(c8.k, c8.v), k, v, slots)
        refuse(ValueError, "k_scales must be", write, ops.KVCache(c8.k, c8.v, t(5, 16, 3, dtype=f32), c8.v_scales), k, v, slots)
        refuse(ValueError, "one shape", write, ops.KVCache(c.k, t(5, 16, 2, 32)), k, v, slots)
        refuse(TypeError, "cache.v", write, ops.KVCache(c.k, c8.v), k, v, slots)
        refuse(ValueError, "k must be", write, c, t(4, 3, 64), v, slots)
        refuse(ValueError, "v must be", write, c, k, t(3, 2, 64), slots)
        refuse(TypeError, "v must be", write, c, k, t(4, 2, 64, dtype=f32), slots)
        refuse(TypeError, "slots", write, c, k, v, t(4, dtype=f32))
        refuse(ValueError, "at most 512", write, ops.KVCache(t(5, 16, 2, 520), t(5, 16, 2, 520)), t(4, 2, 520), t(4, 2, 520), slots)
        refuse(ValueError, "2\\^31", write, ops.KVCache(*(t(1, 1, 2, 64).expand(1 << 20, 1 << 11, 2, 64) for _ in range(2))), k, v, slots)
        refuse(TypeError, "dtype", read, c8, slots, dtype=torch.int8)
        refuse(ValueError, "slots must have 1", read, c, t(4, 1, dtype=i32))
        refuse(TypeError, "dtype", ops.kv_cache, 1, 1, 1, 1, dtype=torch.float64)
        refuse(ValueError, "positive", ops.kv_cache, 0, 1, 1, 1)

        att, table, lens = ops.paged_attention, t(4, 3, dtype=i32), t(4, dtype=i32)
        refuse(TypeError, "q must be", att, t(4, 8, 64, dtype=f32), c, table, lens)
        refuse(TypeError, "does not go with", att, t(4, 8, 64, dtype=torch.float16), c, table, lens)
        refuse(ValueError, "do not go with", att, t(4, 7, 64), c, table, lens)
        refuse(ValueError, "do not go with", att, t(4, 8, 32), c, table, lens)
        refuse(ValueError, "do not go with", att, q, ops.KVCache(t(5, 16, 0, 64), t(5, 16, 0, 64)), table, lens)
        refuse(ValueError, "16 bytes", att, t(4, 8, 72), ops.KVCache(*(t(5, 16, 2, 72, dtype=torch.int8) for _ in range(2)), *c8[2:]), table, lens)
        refuse(ValueError, "at most 256", att, t(4, 8, 264), ops.KVCache(t(5, 16, 2, 264), t(5, 16, 2, 264)), table, lens)
        refuse(ValueError, "4 rows", att, q, c, t(5, 3, dtype=i32), lens)
        refuse(ValueError, "4 rows", att, q, c, table, t(3, dtype=i32))
        refuse(TypeError, "page_table", att, q, c, t(4, 3, dtype=torch.int64), lens)
        refuse(ValueError, "at least 1", att, q, c, t(4, 0, dtype=i32), lens)
        refuse(ValueError, "window", att, q, c, table, lens, window=-1)
        refuse(ValueError, "out must be", att, q, c, table, lens, out=t(4, 8, 32))

        lora, x, y, A, B, ids = ops.lora_add, t(6, 32), t(6, 48), t(3, 8, 32), t(3, 48, 8), t(6, dtype=i32)
        refuse(ValueError, "go together", lora, y, t(6, 31), A, B, ids)
        refuse(ValueError, "go together", lora, y, x, A, t(3, 48, 7), ids)
        refuse(TypeError, "B must be", lora, y, x, A, t(3, 48, 8, dtype=f32), ids)
        refuse(ValueError, "rank", lora, y, x, t(3, 129, 32), t(3, 48, 129), ids)
        refuse(ValueError, "contiguous", lora, y, x, t(3, 32, 8).transpose(1, 2), B, ids)
        refuse(ValueError, "adapters must have", lora, y, x, A, B, t(5, dtype=i32))
        refuse(TypeError, "scales", lora, y, x, A, B, ids, t(3))
        refuse(ValueError, "out must be", lora, y, x, A, B, ids, None, t(6, 47))
        refuse(RuntimeError, "forward only", lora, y, x, A.clone().requires_grad_(), B, ids)


def test_launchers_refuse_what_the_kernels_do_not_take(C):
    """The native entry points check by themselves, before any launch."""
    k = C.kernels
    st4, st12, c4 = [64] * 4, [64] * 12, [16] * 4
    with pytest.raises(ValueError, match="even"):
        k.qk_norm_rope(16, 16, 16, 16, 0, 0, False, [1] * 8, 4, 2, 2, 7, 2, 16, 0, 16, 0, 2, False, 1e-6, 0)
    with pytest.raises(ValueError, match="element type"):
        k.qk_norm_rope(16, 16, 16, 16, 0, 0, False, [1] * 8, 4, 2, 2, 8, 9, 16, 0, 16, 0, 2, False, 1e-6, 0)
    for fn in (k.kv_cache_write, k.kv_cache_read):
        with pytest.raises(ValueError, match="scales"):
            fn([16, 16], st4, 2, [16, 16, 0, 0], st12, 4, 2, 16, 16, 0, 4, 2, 64, 0)
        with pytest.raises(ValueError, match="dim"):
            fn([16, 16], st4, 2, c4, st12, 2, 2, 16, 16, 0, 4, 2, 513, 0)
        with pytest.raises(ValueError, match="sizes"):
            fn([16, 16], st4, 2, c4, st12, 2, 2, 0, 16, 0, 4, 2, 64, 0)
    att = [16, 64, 64, 2, c4, st12, 2, 5, 16, 16, 3, 3, 16, 4, 2, 4, 64, 0, 1.0, 16, 0, 16, 1 << 20, 0]

    def changed(i, v):
        return att[:i] + [v] + att[i + 1:]

    for i, v, match in ((16, 12, "16 bytes"), (4, [8] * 4, "multiples of 16"), (5, [3] * 12, "multiples of 16"), (22, 10, "workspace"),
                        (13, 0, "sizes"), (11, 0, "sizes"), (7, 0, "sizes"), (8, 0, "sizes"), (11, 1 << 30, "2\\^30")):
        with pytest.raises(ValueError, match=match):
            k.paged_attention(*changed(i, v))
    with pytest.raises(ValueError, match="rank"):
        k.lora_add(16, 8, 16, 8, 16, 8, 16, 16, 16, 0, 0, 4, 8, 8, 129, 1, 2, 16, 1 << 20, 0)
    with pytest.raises(ValueError, match="workspace"):
        k.lora_add(16, 8, 16, 8, 16, 8, 16, 16, 16, 0, 0, 4, 8, 8, 16, 1, 2, 16, 1, 0)
