"""Calls of the token-serving operators (seldon_core_amd.ops) that a user can make beside the ordinary ones: what
importing them costs, what is refused, where they are captured, and values at the ends of the types."""
import math
import os
import subprocess
import sys

import pytest
import torch

from seldon_core_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_importing_ops_does_not_load_torch():
    """A CPU component that takes ``crop_resize_chw_ref`` from ops needs numpy only; the token operators come with their first use."""
    code = ("import sys, seldon_core_amd.ops as ops; from seldon_core_amd.ops import crop_resize_chw_ref\n"
            "assert 'torch' not in sys.modules\n"
            "from seldon_core_amd.ops import KVCache, lora_add\n"
            "assert ops.lora_add is lora_add is ops.token_step.lora_add and ops.KVCache is KVCache\n"
            "assert {'kv_cache', 'kv_cache_read', 'kv_cache_write', 'paged_attention', 'qk_norm_rope'} <= set(dir(ops))\n"
            "try:\n    ops.no_such_op\nexcept AttributeError:\n    print('fine')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr


# ---------------------------------------------------------------- refusals
@pytest.fixture
def no_device(monkeypatch):
    """Calls get as far as the native launchers, which refuse before they launch, on a machine without a GPU too."""
    monkeypatch.setattr(ops.token_step, "_stream_of", lambda index: 0)
    monkeypatch.setattr(ops.token_step, "_current_device", lambda: 0)


def fake(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def fake_calls(dtype=torch.bfloat16):
    """One call of each operator on tensors that take part in nothing, as (name, function)."""
    i32, f32, c8 = torch.int32, torch.float32, torch.int8
    q, k, table, n = fake(4, 8, 64, dtype=dtype), fake(4, 2, 64, dtype=dtype), fake(4, 3, dtype=i32), fake(4, dtype=i32)
    cache = ops.KVCache(fake(5, 16, 2, 64, dtype=dtype), fake(5, 16, 2, 64, dtype=dtype))
    eight = ops.KVCache(*(fake(5, 16, 2, 64, dtype=c8) for _ in range(2)), *(fake(5, 16, 2, dtype=f32) for _ in range(2)))
    x, y, A, B = fake(6, 32, dtype=dtype), fake(6, 48, dtype=dtype), fake(3, 8, 32, dtype=dtype), fake(3, 48, 8, dtype=dtype)
    return {
        "rope": lambda: ops.qk_norm_rope(q, k, None, None, n, fake(32, dtype=f32)),
        "write": lambda: ops.kv_cache_write(cache, k, k.clone(), n),
        "write 8": lambda: ops.kv_cache_write(eight, k, k.clone(), n),
        "read": lambda: ops.kv_cache_read(cache, n),
        "read 8": lambda: ops.kv_cache_read(eight, n),
        "attention": lambda: ops.paged_attention(q, cache, table, n, return_lse=True),
        "attention 8": lambda: ops.paged_attention(q, eight, table, n),
        "lora": lambda: ops.lora_add(y, x, A, B, fake(6, dtype=i32), fake(3, dtype=f32)),
    }


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
@pytest.mark.parametrize("op", ["rope", "write", "write 8", "read", "read 8", "attention", "attention 8", "lora"])
def test_fake_tensors_are_refused(op, no_device):
    """Every check of shapes and types holds for a fake tensor, whose address is 0: no kernel may be given it."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        call = fake_calls()[op]
        with pytest.raises(ValueError, match="no memory|has scales"):
            call()


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_a_fake_weight_is_not_taken_for_none():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        w = fake(64)
    assert ops.token_step._optional(None, "w") == 0
    with pytest.raises(ValueError, match="w has no memory"):
        ops.token_step._optional(w, "w")


def test_launchers_refuse_null_pointers(C):
    k = C.kernels
    st4, st12, c4 = [64] * 4, [64] * 12, [16] * 4
    rope = [16, 16, 16, 16, 0, 0, False, [1] * 8, 4, 2, 2, 8, 2, 16, 0, 16, 0, 2, False, 1e-6, 0]
    cache = [[16, 16], st4, 2, c4, st12, 2, 2, 16, 16, 0, 4, 2, 64, 0]
    att = [16, 64, 64, 2, c4, st12, 2, 5, 16, 16, 3, 3, 16, 4, 2, 4, 64, 0, 1.0, 16, 0, 16, 1 << 20, 0]
    lora = [16, 8, 16, 8, 16, 8, 16, 16, 16, 0, 0, 4, 8, 8, 16, 1, 2, 16, 1 << 20, 0]
    for fn, args, at in ((k.qk_norm_rope, rope, (0, 1, 2, 3, 13, 15)), (k.kv_cache_write, cache, (8,)), (k.kv_cache_read, cache, (8,)),
                         (k.paged_attention, att, (0, 9, 12, 19, 21)), (k.lora_add, lora, (0, 2, 4, 6, 7, 8, 17))):
        for i in at:
            with pytest.raises(ValueError, match="no memory"):
                fn(*args[:i], 0, *args[i + 1:])
    for rows, c in (([16, 0], c4), ([0, 16], c4), ([16, 16], [16, 0, 0, 0]), ([16, 16], [0, 16, 0, 0])):
        with pytest.raises(ValueError, match="no memory"):
            k.kv_cache_write(rows, st4, 2, c, *cache[4:])
    with pytest.raises(ValueError, match="no memory"):
        k.paged_attention(*att[:4], [16, 0, 0, 0], *att[5:])


def test_gradients_of_both_modes_are_refused():
    """Reverse mode by requires_grad, forward mode by a tangent (whose tensor does not require a gradient); the scales of an 8-bit
    cache too."""
    import torch.autograd.forward_ad as fw
    from torch._subclasses.fake_tensor import FakeTensorMode

    f32, i32 = torch.float32, torch.int32
    with FakeTensorMode():
        q, k, n, inv = fake(4, 8, 64, dtype=f32), fake(4, 2, 64, dtype=f32), fake(4, dtype=i32), fake(32, dtype=f32)
        x, y, A, B, ids = fake(6, 32, dtype=f32), fake(6, 48, dtype=f32), fake(3, 8, 32, dtype=f32), fake(3, 48, 8, dtype=f32), fake(6, dtype=i32)
        qh, table = fake(4, 8, 64), fake(4, 3, dtype=i32)

        def eight(f):
            s = fake(5, 16, 2, dtype=f32)
            return ops.KVCache(*(fake(5, 16, 2, 64, dtype=torch.int8) for _ in range(2)), s.clone(), f(s))

        def calls(f):
            return {
                "q": lambda: ops.qk_norm_rope(f(q), k, None, None, n, inv),
                "k": lambda: ops.qk_norm_rope(q, f(k), None, None, n, inv),
                "q_weight": lambda: ops.qk_norm_rope(q, k, f(fake(64, dtype=f32)), None, n, inv),
                "inv_freq": lambda: ops.qk_norm_rope(q, k, None, None, n, f(inv)),
                "v": lambda: ops.kv_cache_write(ops.KVCache(fake(5, 16, 2, 64), fake(5, 16, 2, 64)), k, f(k.clone()), n),
                "cache.v_scales": lambda: ops.kv_cache_read(eight(f), n),
                " cache.v_scales": lambda: ops.paged_attention(qh, eight(f), table, n),
                "y": lambda: ops.lora_add(f(y), x, A, B, ids),
                "x": lambda: ops.lora_add(y, f(x), A, B, ids),
                "B": lambda: ops.lora_add(y, x, A, f(B), ids),
                "scales": lambda: ops.lora_add(y, x, A, B, ids, f(fake(3, dtype=f32))),
            }

        for name, call in calls(lambda t: t.clone().requires_grad_()).items():
            with pytest.raises(RuntimeError, match=f"^{name.strip()} requires a gradient"):
                call()
        with fw.dual_level():
            for name, call in calls(lambda t: fw.make_dual(t, torch.ones_like(t))).items():
                with pytest.raises(RuntimeError, match=f"^{name.strip()} has a tangent"):
                    call()


def test_views_whose_sign_is_put_off_are_refused():
    """torch.conj(z).imag holds z's own numbers and a flag that says "negated", which a kernel does not see."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    f32, i32 = torch.float32, torch.int32
    assert torch.ones(2, dtype=torch.complex64).conj().imag.is_neg()
    with FakeTensorMode():
        q = fake(4, 8, 1, dtype=torch.complex64).conj().imag  # a last dimension of one: any stride goes
        assert q.is_neg()
        with pytest.raises(ValueError, match="k is a view whose sign"):
            ops.kv_cache_write(ops.KVCache(fake(5, 16, 8, 1), fake(5, 16, 8, 1)), q, fake(4, 8, 1, dtype=f32), fake(4, dtype=i32))
        s = fake(5, 16, 2, dtype=torch.complex64).conj().imag
        c = ops.KVCache(*(fake(5, 16, 2, 64, dtype=torch.int8) for _ in range(2)), fake(5, 16, 2, dtype=f32), s)
        with pytest.raises(ValueError, match="cache.v_scales is a view whose sign"):
            ops.kv_cache_read(c, fake(4, dtype=i32))


def test_calls_too_large_for_a_launch_are_refused_whole(C):
    """A launch has fewer than 2^32 threads along x: what would need more is refused before the first launch."""
    k = C.kernels
    st4, st12, c4 = [64] * 4, [64] * 12, [16] * 4
    with pytest.raises(ValueError, match="too large"):  # 2^26 tokens, 4 a workgroup of 256 threads
        k.qk_norm_rope(16, 16, 16, 16, 0, 0, False, [1] * 8, 1 << 26, 2, 2, 8, 2, 16, 0, 16, 0, 2, False, 1e-6, 0)
    for fn in (k.kv_cache_write, k.kv_cache_read):  # dim 512: a wave for each of 2^26 heads
        with pytest.raises(ValueError, match="too large"):
            fn([16, 16], st4, 2, c4, st12, 2, 2, 16, 16, 0, 1 << 23, 8, 512, 0)
    with pytest.raises(ValueError, match="too large"):  # 2^18 requests of 64 heads: a workgroup each to join their parts
        k.paged_attention(16, 64, 64, 2, c4, st12, 2, 5, 16, 16, 16, 16, 16, 1 << 18, 8, 8, 64, 0, 1.0, 16, 0, 16, 1 << 40, 0)
    with pytest.raises(ValueError, match="too large"):  # 2^28 rows, 32 a workgroup of 512 threads
        k.lora_add(16, 8, 16, 8, 16, 8, 16, 16, 16, 0, 0, 1 << 28, 8, 8, 16, 1, 2, 16, 1 << 50, 0)


# --------------------------------------------------------- values at the ends
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHE = {"same": None, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_paged_attention_scores_as_large_as_the_types_give(dtype, cache):
    """Scores of 2^20 to 2^29, a few ulps apart, where fp32 has no room for the distance that weights are kept at.

    All tokens hold the same value, so whatever the weights are, the output is that value: weights that are split, w (1 +- 2^-16), and
    n + 64 fp32 roundings of the sums, and one rounding to the type."""
    g, dt, n, D = gen(3), DT[dtype], 700, 64
    for power in range(20, 30):
        c = ops.kv_cache(-(-n // 16), 16, 1, D, dtype=CACHE[cache] or dt)
        k = torch.zeros((n, 1, D))
        k[:, 0, 0] = 2.0 ** (power - 14)
        k[:, 0, 1] = torch.randint(0, 200, (n,), generator=g) if cache == "same" else 0
        k[:, 0, 0] *= 1 if cache == "same" else 1 + torch.randint(0, 2, (n,), generator=g) / 8  # steps that e4m3 has
        # 8 bits hold powers of two exactly, under whatever scale
        value = torch.tensor([1.0, -2.0, 0.5, 0.25, 0.0, 1.0, -1.0, -0.125]).repeat(D // 8) if cache != "same" else randn(g, D, dtype=dt).float()
        v = value.expand(n, 1, D)
        ops.kv_cache_write(c, k.to(dt).cuda(), v.to(dt).cuda(), torch.arange(n).cuda())
        q = torch.zeros((1, 2, D), dtype=dt)
        q[..., 0], q[..., 1] = 2.0 ** 14, 1
        table, lens = torch.arange(-(-n // 16)).int()[None].cuda(), torch.tensor([n]).int().cuda()
        out, lse = ops.paged_attention(q.cuda(), c, table, lens, scale=1.0, return_lse=True)
        rel = torch.finfo(dt).eps / 2 + 2.0 ** -16 + (n + 64) * 2.0 ** -24
        assert bool(((out.cpu().double() - value.double()).abs() <= rel * value.abs().double()).all()), f"2^{power}: {out[0, 0, :4]}"
        s = k[:, 0, 0].double() * 2.0 ** 14 + k[:, 0, 1].double()
        # the products' sum, its product with log2(e), and the way back: a few roundings of the score
        assert bool(((lse.cpu().double() - torch.logsumexp(s, 0)).abs() <= 4 * 2.0 ** -24 * float(s.max()) + 1e-4).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_paged_attention_values_that_are_not_finite(dtype, cache):
    """One token's value of a request is infinite or NaN.  Seen, the dimension it is in (with 8 bits, which keep one scale for the
    head: the head) is not finite, however small the token's weight; outside of the window it does not matter."""
    g, dt, n, H, D = gen(4), DT[dtype], 300, 2, 64
    for bad in (math.inf, -math.inf, math.nan):
        for depth in (0.0, 2.0, 400.0):  # the token's score below the others: its weight is ordinary, small, or 0 in fp32
            c = ops.kv_cache(-(-n // 16), 16, H, D, dtype=CACHE[cache] or dt)
            k, v = 0.1 * randn(g, n, H, D), randn(g, n, H, D)
            k[..., 0] = 1
            k[100, 1, 0] = 1 - depth / 8
            v[100, 1, 7] = bad
            q = 0.1 * randn(g, 1, 2 * H, D)
            q[..., 0] = 8
            ops.kv_cache_write(c, k.to(dt).cuda(), v.to(dt).cuda(), torch.arange(n).cuda())
            table, lens = torch.arange(-(-n // 16)).int()[None].cuda(), torch.tensor([n]).int().cuda()
            out, lse = (x.cpu() for x in ops.paged_attention(q.to(dt).cuda(), c, table, lens, scale=1.0, return_lse=True))
            assert torch.isfinite(out[:, :2]).all() and torch.isfinite(lse).all()
            hit = torch.zeros(D, dtype=torch.bool)
            hit[7] = True
            if cache != "same":
                hit[:] = True
            assert not torch.isfinite(out[:, 2:, hit]).any(), (bad, depth, out[0, 2, :8])
            assert torch.isfinite(out[:, 2:, ~hit]).all()
            if cache != "same" or math.isnan(bad):
                assert out[:, 2:, hit].isnan().all()
            out = ops.paged_attention(q.to(dt).cuda(), c, table, lens, scale=1.0, window=n - 101)
            assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 700])
@pytest.mark.parametrize("dtype", list(DT))
def test_lora_add_weights_that_are_not_finite(dtype, T):
    """An infinite or NaN weight of B reaches its own column of its own adapter's rows, and one of A all columns of them."""
    g, dt = gen(5), DT[dtype]
    K, M, r, N = 96, 130, 12, 3
    x, y = randn(g, T, K, dtype=dt), randn(g, T, M, dtype=dt)
    A, B = (randn(g, N, r, K) * 0.1).to(dt), randn(g, N, M, r, dtype=dt)
    ids = (torch.arange(T) * 7 % (N + 1)).int()  # N: none
    hit = ids == 1
    for bad in (math.inf, -math.inf, math.nan):
        b = B.clone()
        b[1, 70, 11] = bad
        got = ops.lora_add(y.cuda(), x.cuda(), A.cuda(), b.cuda(), ids.cuda()).cpu()
        assert not torch.isfinite(got[hit][:, 70]).any()
        if dtype == "fp32" and not math.isnan(bad):  # h in one piece: the formula's own infinity
            sign = torch.sign(x[hit].double() @ A[1, 11].double())
            assert torch.equal(got[hit][:, 70].double(), sign * bad)
        a = A.clone()
        a[1, 11, 95] = bad
        some = ops.lora_add(y.cuda(), x.cuda(), a.cuda(), B.cuda(), ids.cuda()).cpu()
        assert not torch.isfinite(some[hit]).any()
        for o, keep in ((got, torch.ones(M, dtype=torch.bool)), (some, torch.ones(M, dtype=torch.bool))):
            assert torch.isfinite(o[~hit]).all() and torch.equal(o[ids == N], y[ids == N])
        cols = torch.arange(M) != 70
        assert torch.isfinite(got[:, cols]).all()


# ------------------------------------------------------------- captured calls
class CacheStep(torch.nn.Module):
    """Rows of [slot, values]: writes each row's key and value at its slot, and gives back what the cache then holds there."""

    def __init__(self, cache):
        super().__init__()
        self.cache = cache

    def forward(self, x):
        slots, k = x[:, 0].long(), x[:, 1:].reshape(len(x), *self.cache.k.shape[2:])
        ops.kv_cache_write(self.cache, k, 2 * k, slots)
        k, v = ops.kv_cache_read(self.cache, slots)
        return k.flatten(1) + v.flatten(1)


@pytest.mark.gpu
def test_graphed_module_leaves_a_cache_to_its_rows():
    """GraphedModule runs a module on zeros before it captures it, and pads batches with zeros: rows that would be written at slot 0
    of a live request.  A module that writes a cache is served eagerly, each row once."""
    from seldon_core_amd.models.graphed import GraphedModule

    cache = ops.kv_cache(4, 4, 2, 8, dtype=torch.float32)
    live = torch.full((1, 2, 8), 5.0, device="cuda")
    ops.kv_cache_write(cache, live, live, torch.zeros(1, dtype=torch.int64, device="cuda"))
    m = GraphedModule(CacheStep(cache), max_batch=8)
    g = gen(6)
    for n in (3, 11, 5):  # buckets of 4, 8 + 4 and 8
        x = randn(g, n, 17)
        x[:, 0] = 1 + torch.randperm(15, generator=g)[:n]
        out = m(x.numpy())
        assert torch.equal(torch.from_numpy(out), 3 * x[:, 1:])
        assert torch.equal(cache.k[0, 0], live[0]) and torch.equal(cache.v[0, 0], live[0])
    assert "cache" in m.graph_error and m.replays == 0 and m.eager_calls == 4

    class Reader(torch.nn.Module):  # what only reads is captured
        def forward(self, x):
            k, _ = ops.kv_cache_read(cache, x[:, 0].long())
            return k.flatten(1)

    r = GraphedModule(Reader(), max_batch=8)
    x = torch.zeros(3, 1)
    assert torch.equal(torch.from_numpy(r(x.numpy())), live.flatten(1).cpu().expand(3, 16)) and r.graph_error is None and r.replays == 1


def test_a_cache_is_not_written_in_a_rehearsal():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        cache, k = ops.KVCache(fake(5, 16, 2, 64), fake(5, 16, 2, 64)), fake(0, 2, 64)
        write = lambda: ops.kv_cache_write(cache, k, k, fake(0, dtype=torch.int32))  # noqa: E731
        assert write() is cache
        with ops.token_step.no_cache_writes("rows of zeros"):
            with pytest.raises(RuntimeError, match="rows of zeros"):
                write()
        assert write() is cache


@pytest.mark.gpu
def test_a_step_on_a_side_stream_waits_for_its_inputs():
    """The block of test_decoder_ops on a stream of its own, while the default stream has yet to make its inputs: it orders itself
    behind them.  (Either way every index is a valid one: the inputs hold an earlier step's.)"""
    from test_decoder_ops import Step, step_inputs

    T, page, W, Hq, H, D, tenants = 5, 16, 4, 8, 2, 64, 3
    g = gen(21)
    m = Step(256, Hq, H, D, tenants, T * W, page, torch.bfloat16, g)
    table = torch.randperm(T * W, generator=g).int().view(T, W).cuda()
    old, new = (step_inputs(g, T, tenants, W, page, 3 + 20 * i) for i in range(2))
    with torch.no_grad():
        m(*old, table)
        want = m(*new, table).clone()
        for c in m.cache[:2]:
            c.zero_()
        m(*old, table)
        sx, st, sp = (t.clone() for t in old)
        side, a = torch.cuda.Stream(), torch.randn(8192, 8192, device="cuda")
        torch.cuda.synchronize()
        for _ in range(5):  # tens of milliseconds in front of the inputs
            a @ a
        for s, n in zip((sx, st, sp), new):
            s.copy_(n)
        with torch.cuda.stream(side):
            got = m(sx, st, sp, table)
        torch.cuda.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------- adapters: the larger forms
def lora_check(got, y, x, A, B, ids, scales):
    """As test_decoder_ops has it: two sums in fp32 ((K + r + 8) 2^-24 of the sum of magnitudes), h in two 16-bit parts (2^-16 of it
    in bf16, 2^-24 of the row's largest h in fp16, whose remainder may be subnormal), one rounding to the type."""
    from test_decoder_ops import close

    (N, r, K), dt = A.shape, x.dtype
    want, mag = ops.token_step.lora_add_ref(y, x, A, B, ids, scales)
    atol = (K + r + 8) * 2.0 ** -24 * mag + (2.0 ** -16 * mag if dt == torch.bfloat16 else 0)
    if dt == torch.float16:
        for a in range(N):
            rows = ids == a
            h = (x[rows].double() @ A[a].double().T).abs().amax(-1, keepdim=True) * (1.0 if scales is None else abs(scales[a].double()))
            atol[rows] += 2.0 ** -23 * h * B[a].double().abs().sum(-1)
    close(got, want, dt, atol + 2.0 ** -24 * want.abs())
    none = (ids < 0) | (ids >= N)
    assert torch.equal(got.cpu()[none], y[none])


LORA = [  # rows, inner, outer, rank, adapters, mixed: many rows of uneven ranks, one and several column tiles of a workgroup, ends inside
    (1500, 200, 1100, 12, 6, True), (1500, 72, 3000, 13, 6, True), (700, 130, 330, 27, 5, True), (1300, 130, 3300, 27, 4, False),
    (300, 136, 1503, 99, 4, True), (900, 136, 5000, 99, 3, True), (2000, 96, 2100, 9, 3, False), (400, 200, 1000, 77, 3, True),
    (330, 96, 640, 100, 5, True), (400, 160, 700, 128, 3, False), (300, 64, 4000, 50, 2, True),
    # four rows of a workgroup, several column tiles
    (512, 100, 1100, 8, 6, True), (120, 64, 5000, 64, 4, True), (130, 72, 6000, 27, 3, True), (64, 64, 9000, 101, 2, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LORA, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", list(DT))
def test_lora_add_larger_forms(case, dtype):
    T, K, M, r, N, mixed = case
    g, dt = gen(sum(case)), DT[dtype]
    x, y = randn(g, T, K, dtype=dt), randn(g, T, M, dtype=dt)
    A, B, scales = (randn(g, N, r, K) * K ** -0.5).to(dt), (randn(g, N, M, r) * r ** -0.5).to(dt), randn(g, N)
    ids = torch.randint(-1, N + 1, (T,), generator=g) if mixed else torch.arange(T) * N // T
    ids[-1] = N - 1  # the last adapter's last run, with nothing behind it
    got = ops.lora_add(y.cuda(), x.cuda(), A.cuda(), B.cuda(), ids.cuda(), scales.cuda())
    lora_check(got, y, x, A, B, ids, scales)


@pytest.mark.gpu
def test_lora_add_sorted_rows_in_a_captured_graph():
    """A large mixed batch, sorted by a launch of its own: replays with other rows and adapters, with eager calls in between, give
    what eager calls give; one of the replays has its rows in runs, which leaves the sort out."""
    g = gen(7)
    T, K, M, r, N = 900, 128, 192, 16, 40
    A, B = ((randn(g, *s) * 0.1).bfloat16() for s in ((N, r, K), (N, M, r)))
    steps = [(randn(g, T, K, dtype=torch.bfloat16), randn(g, T, M, dtype=torch.bfloat16), torch.randint(-1, N, (T,), generator=g)) for _ in range(4)]
    steps[2][2].copy_(torch.sort(steps[2][2]).values // 4)
    Ad, Bd = A.cuda(), B.cuda()
    static = [t.cuda() for t in steps[0]]
    graph = torch.cuda.CUDAGraph()
    ops.lora_add(static[1], static[0], Ad, Bd, static[2])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.lora_add(static[1], static[0], Ad, Bd, static[2])
    for x, y, ids in steps:
        for s, t in zip(static, (x, y, ids)):
            s.copy_(t)
        graph.replay()
        eager = ops.lora_add(static[1], static[0], Ad, Bd, static[2])
        other = ops.lora_add(static[1], static[0], Ad, Bd, (static[2] + 1) % N)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and not torch.equal(out, other)
        lora_check(out, y, x, A, B, ids, None)


# ------------------------------------------------------------ what is written
def test_tensors_that_hold_an_element_twice_are_not_written():
    """An expanded out or cache names the same memory for several rows, which kernels would write in any order."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    f32, i32 = torch.float32, torch.int32
    with FakeTensorMode():
        q, k, n, inv = fake(4, 8, 64), fake(4, 2, 64), fake(4, dtype=i32), fake(32, dtype=f32)
        x, y, A, B, ids = fake(6, 32), fake(6, 48), fake(3, 8, 32), fake(3, 48, 8), fake(6, dtype=i32)
        pages = fake(1, 16, 2, 64).expand(5, 16, 2, 64)
        c8 = [fake(5, 16, 2, 64, dtype=torch.int8) for _ in range(2)]
        for name, call in {
            r"out\[1\]": lambda: ops.qk_norm_rope(q, k, None, None, n, inv, out=(q, fake(4, 1, 64).expand(4, 2, 64))),
            "cache.k": lambda: ops.kv_cache_write(ops.KVCache(pages, fake(5, 16, 2, 64)), k, k, n),
            "cache.v": lambda: ops.kv_cache_write(ops.KVCache(fake(5, 16, 2, 64), pages), k, k, n),
            "cache.k_scales": lambda: ops.kv_cache_write(ops.KVCache(*c8, fake(5, 16, 1, dtype=f32).expand(5, 16, 2), fake(5, 16, 2, dtype=f32)), k, k, n),
            "out": lambda: ops.lora_add(y, x, A, B, ids, out=fake(1, 48).expand(6, 48)),
        }.items():
            with pytest.raises(ValueError, match=f"^{name} holds elements more than once"):
                call()
        # a dimension of one has any stride
        one = fake(1, 48).as_strided((1, 48), (0, 1))
        assert ops.token_step._written(one, "out") is None


@pytest.mark.gpu
def test_outputs_over_inputs_are_refused():
    """The host sees where tensors lie: an output over an input that other workgroups still read is refused, one in its place (where
    that is allowed) or beside it in one buffer is not."""
    g, bf = gen(8), torch.bfloat16
    buf = randn(g, 40, 256, dtype=bf).cuda()
    y, x, out = buf[:8], buf[8:16], buf[4:12]
    A, B, ids = randn(g, 2, 8, 256, dtype=bf).cuda(), randn(g, 2, 256, 8, dtype=bf).cuda(), torch.zeros(8, dtype=torch.int32, device="cuda")
    for o in (x, out):
        with pytest.raises(ValueError, match="out lies over"):
            ops.lora_add(y, x, A, B, ids, out=o)
    with pytest.raises(ValueError, match="out lies over y"):  # the same first element, other rows
        ops.lora_add(buf.view(20, 512)[:8, :256], buf[30:38], A, B, ids, out=buf[:8])
    with pytest.raises(ValueError, match="out lies over y"):  # a row further
        ops.lora_add(y, x, A, B, ids, out=buf[1:9])
    want = ops.lora_add(y, x, A, B, ids)
    assert torch.equal(ops.lora_add(y, x, A, B, ids, out=buf[16:24]), want)
    wide = buf[24:32].reshape(4, 512).repeat(2, 1)
    a, b = wide[:, :256], wide[:, 256:]
    want = ops.lora_add(a, b, A, B, ids)
    assert torch.equal(ops.lora_add(a, b, A, B, ids, out=a), want)  # side by side in one buffer, and in place

    T, D = 4, 64
    pos, inv = torch.arange(T, device="cuda"), torch.ones(32, device="cuda")
    q, k = (randn(g, T, 2, D, dtype=bf).cuda() for _ in range(2))
    for o in ((k, q), (q, q), (k, torch.empty_like(k))):
        with pytest.raises(ValueError, match="lies over"):
            ops.qk_norm_rope(q, k, None, None, pos, inv, out=o)
    both = torch.cat((q, k), 1)
    want = ops.qk_norm_rope(q, k, None, None, pos, inv)
    got = ops.qk_norm_rope(both[:, :2], both[:, 2:], None, None, pos, inv, out=(both[:, :2], both[:, 2:]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c = ops.kv_cache(4, 4, 2, D)
    with pytest.raises(ValueError, match="out lies over q"):
        ops.paged_attention(q, c, torch.zeros((T, 1), dtype=torch.int32, device="cuda"), pos.int(), out=q)
    e = torch.empty((0, 2, D), dtype=bf, device="cuda")
    assert ops.qk_norm_rope(e, e, None, None, pos[:0], inv, out=(e, e))[0] is e  # nothing lies over nothing


@pytest.mark.gpu
def test_writes_are_counted_for_autograd():
    """What an op of autograd's kept for its backward pass and an operator then writes over raises there, as with torch's own."""
    g = gen(9)
    x, A, B = randn(g, 3, 8).cuda(), randn(g, 1, 4, 8).cuda(), randn(g, 1, 8, 4).cuda()
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    w, buf = torch.ones(8, device="cuda", requires_grad=True), torch.zeros((3, 8), device="cuda")
    loss = (w * buf).sum()
    ops.lora_add(buf, x, A, B, ids, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    q, k, pos, inv = randn(g, 3, 2, 8).cuda(), randn(g, 3, 2, 8).cuda(), ids.clone(), torch.ones(4, device="cuda")
    before = q._version, k._version
    ops.qk_norm_rope(q, k, None, None, pos, inv, out=(q, k))
    assert (q._version, k._version) > before and k._version > before[1]
    c = ops.kv_cache(2, 4, 2, 8, dtype=torch.int8)
    before = [t._version for t in c]
    ops.kv_cache_write(c, q, k, torch.arange(3, device="cuda"))
    assert all(t._version > b for t, b in zip(c, before))
    with torch.inference_mode():
        ops.kv_cache_write(ops.kv_cache(2, 4, 2, 8), q, k, torch.arange(3, device="cuda"))


@pytest.mark.gpu
def test_writes_without_gradients_are_counted_too():
    """As torch's own in-place operations are: what was kept may be from outside of the no_grad block."""
    g = gen(9)
    x, A, B = randn(g, 3, 8).cuda(), randn(g, 1, 4, 8).cuda(), randn(g, 1, 8, 4).cuda()
    for without in (torch.no_grad, torch.inference_mode):
        w, buf = torch.ones(8, device="cuda", requires_grad=True), torch.zeros((3, 8), device="cuda")
        loss = (w * buf).sum()
        with without():
            ops.lora_add(buf, x, A, B, torch.zeros(3, dtype=torch.int32, device="cuda"), out=buf)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_a_forced_build_compiles_what_is_there_already(monkeypatch):
    import importlib.util
    import types

    spec = importlib.util.spec_from_file_location("build_native", os.path.join(ROOT, "tools", "build_native.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    ran = []
    monkeypatch.setattr(b, "_needs_build", lambda src, obj: False)
    monkeypatch.setattr(b, "subprocess", types.SimpleNamespace(run=lambda cmd, **kw: ran.append(cmd) or types.SimpleNamespace(returncode=0, stderr="")))
    b._compile("kernels/rope.hip", False)
    assert not ran
    b._compile("kernels/rope.hip", False, force=True)
    assert len(ran) == 1 and "+packed" not in " ".join(ran[0]) and "-packed-fp32-ops" in ran[0]


def test_sizes_of_nothing_are_refused_not_divided_by(C):
    """A cache of pages without slots, and workspaces of no tokens or rows: errors, not a division by zero, which ends the process."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    code = ("import torch\nfrom seldon_core_amd import native\nk = native().kernels\n"
            "for f, a in ((k.paged_attention_workspace, (1, 1, 1, 64, False, 0, 0)), (k.lora_workspace, (0, 64, 8, 1))):\n"
            "    try:\n        f(*a)\n    except ValueError as e:\n        print(e)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.count("sizes") == 2, (r.returncode, r.stdout, r.stderr)
    with FakeTensorMode():
        c = ops.KVCache(fake(5, 0, 2, 64), fake(5, 0, 2, 64))
        with pytest.raises(ValueError, match="at least 1"):
            ops.paged_attention(fake(4, 8, 64), c, fake(4, 3, dtype=torch.int32), fake(4, dtype=torch.int32))


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_a_window_larger_than_any_table_sees_all(no_device, monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensorMode

    seen = []
    monkeypatch.setattr(ops.token_step, "_attention_workspace", lambda *sizes: seen.append(sizes) or 1)
    with FakeTensorMode():
        c, q, table, n = ops.KVCache(fake(5, 16, 2, 64), fake(5, 16, 2, 64)), fake(4, 8, 64), fake(4, 3, dtype=torch.int32), fake(4, dtype=torch.int32)
        for window in (2 ** 40, 48, 47):
            with pytest.raises(ValueError):  # by the launcher, as far as a fake call gets
                ops.paged_attention(q, c, table, n, window=window)
    assert [s[-1] for s in seen] == [48, 48, 47]


@pytest.mark.gpu
def test_a_window_larger_than_any_table_gives_the_same():
    g = gen(10)
    c = ops.kv_cache(20, 16, 2, 64)
    ops.kv_cache_write(c, *(randn(g, 300, 2, 64, dtype=torch.bfloat16).cuda() for _ in range(2)), torch.arange(300, device="cuda"))
    q, table = randn(g, 2, 4, 64, dtype=torch.bfloat16).cuda(), torch.arange(20, device="cuda").int().expand(2, 20)
    n = torch.tensor([300, 77], device="cuda").int()
    assert torch.equal(ops.paged_attention(q, c, table, n, window=2 ** 40), ops.paged_attention(q, c, table, n))


@pytest.mark.gpu
def test_rows_of_the_cache_itself_move_to_other_slots():
    """k and v may be views of the cache that is written, where no row is both read and written."""
    g = gen(11)
    c = ops.kv_cache(6, 16, 3, 64)
    rows = [randn(g, 96, 3, 64, dtype=torch.bfloat16).cuda() for _ in range(2)]
    ops.kv_cache_write(c, *rows, torch.arange(96, device="cuda"))
    ops.kv_cache_write(c, c.k[1], c.v[1], torch.arange(64, 80, device="cuda"))
    k, v = ops.kv_cache_read(c, torch.arange(96, device="cuda"))
    for got, was in ((k, rows[0]), (v, rows[1])):
        want = was.clone()
        want[64:80] = was[16:32]
        assert torch.equal(got, want)
