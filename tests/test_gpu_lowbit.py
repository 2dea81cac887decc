"""`-m gpu`: the low-bit decode step's operators (4-bit linears, the e4m3 key/value cache, next-token scores) against their definitions in 64
bits, written out in plain torch.

Tolerances.  A result rounded once to bf16 is off by at most 2^-8 of its value (half a step).  fp32 sums of n terms are off by at most n 2^-24 of the
sum of their absolute values; the terms are named at each test.  What is defined in fp32 operation by operation (cache codes and
scales, rotated queries, processed scores) has to be equal bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F8, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float64
HALF_BF = 2.0 ** -8


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from physicedit_amd import ops as o
    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def replays(fn, inputs, others, check):
    """captures fn() once on the static `inputs`, replays it on each set of `others` with eager work and synchronisation in between"""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    for new in others:
        for dst, src in zip(inputs, new):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        check(out, fn())


# ---- linears with 4-bit weights ------------------------------------------------------------------------------------------------------------------

def w4_case(g, M, N, K, group, zero):
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda").to(torch.uint8)
    scale = (0.02 * torch.exp(0.5 * randn(g, N, K // group))).to(BF)
    z = torch.randint(0, 16, (N, K // group), generator=g, device="cuda").to(torch.uint8) if zero else None
    return codes, scale, z, randn(g, M, K).to(BF)


def w4_weight(codes, scale, zero, group):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).to(F64)
    z = 8.0 if zero is None else zero.to(F64).repeat_interleave(group, 1)
    return (c - z) * scale.to(F64).repeat_interleave(group, 1)


def w4_reference(w, scale, group, x, eps=None, bias=None, res=None, swiglu=False):
    """-> the result in 64 bits and how far fp32 may be from it.  The kernel sums (128 + code) x and takes (128 + zero) sum x off: terms of at most
    143 |x|, twice, in a chain of `group` per group, then one per group, then the waves: gamma = (group + K / group + 32) 2^-24."""
    xd = x.to(F64)
    K = x.shape[1]
    y = xd @ w.T
    slack = (group + K // group + 32) * 2.0 ** -24 * 286 * (xd.abs() @ scale.to(F64).repeat_interleave(group, 1).T)
    if eps is not None:
        r = 1 / (xd.square().mean(1, keepdim=True) + eps).sqrt()
        y, slack = y * r, slack * r + K * 2.0 ** -24 * (y * r).abs()
    if bias is not None:
        y = y + bias.to(F64)
    if swiglu:
        a, b = y.chunk(2, 1)
        sa, sb = slack.chunk(2, 1)
        y = a * torch.sigmoid(a) * b
        slack = 1.1 * sa * b.abs() + a.abs() * sb + sa * sb + 2.0 ** -20 * y.abs()      # |d silu| <= 1.1; expf and the division: a few 2^-22
    if res is not None:
        y = y + res.to(F64)
    return y, slack


def near(got, want, slack):
    err = (got.to(F64) - want).abs()
    bound = HALF_BF * (want.abs() + slack) + slack + 2.0 ** -130
    assert got.isfinite().all() and (err <= bound).all(), f"off by up to {(err / bound).max().item():.3g} of the bound"
    # every element is within half a bf16 step of something close to the result: so is the whole
    assert err.norm() <= HALF_BF * want.norm() + slack.norm() * 0.1 + 1e-30


@pytest.mark.parametrize("M,N,K,group,zero,norm,bias,res,swiglu", [
    (1, 1, 32, 32, True, False, False, False, False),
    (1, 16, 128, 128, False, True, True, True, False),
    (1, 33, 416, 32, True, True, True, False, False),
    (1, 4608, 3584, 128, True, True, True, False, False),
    (1, 3584, 18944, 128, True, False, False, True, False),
    (2, 1000, 3584, 64, True, False, True, True, False),
    (5, 151, 320, 64, False, True, False, True, False),
    (16, 48, 1152, 128, True, True, True, True, False),
    (17, 47, 160, 32, True, True, True, True, False),
    (32, 130, 2048, 64, True, False, False, False, False),
    (33, 501, 1056, 32, False, True, True, True, False),
    (64, 77, 1920, 128, True, True, True, True, False),
    (64, 3000, 96, 32, True, False, True, False, False),
    (3, 20000, 256, 128, True, False, False, True, False),
    (1, 32, 64, 64, True, True, True, False, True),
    (1, 37888, 3584, 128, True, True, False, False, True),
    (7, 160, 192, 64, False, False, True, False, True),
    (20, 352, 1056, 32, True, True, True, False, True),
    (64, 96, 640, 128, True, True, True, False, True)])
def test_gemv_w4(ops, M, N, K, group, zero, norm, bias, res, swiglu):
    g = gen(M * 1000 + N)
    codes, scale, z, x = w4_case(g, M, N, K, group, zero)
    b = randn(g, N).to(BF) if bias else None
    r = randn(g, M, N).to(BF) if res else None
    got = ops.gemv_w4(x, ops.pack_w4(codes, scale, z, group), bias=b, res=r, epilogue="swiglu" if swiglu else "bias", norm_eps=1e-6 if norm else None)
    want, slack = w4_reference(w4_weight(codes, scale, z, group), scale, group, x, 1e-6 if norm else None, b, r, swiglu)
    assert got.shape == want.shape and got.dtype == BF
    near(got, want, slack)


@pytest.mark.parametrize("M", [1, 8, 16, 20, 33, 60])
@pytest.mark.parametrize("N", [1888, 8096, 12064, 17504])          # 118, 506, 754, 1094 tiles of 16: each side of the rules on their number
@pytest.mark.parametrize("group", [32, 64, 128])
def test_gemv_w4_variants(ops, M, N, group):
    """every kernel that the rules on sizes choose, with more chunks of 128 inputs than waves and the last one cut short"""
    g = gen(M * N + group)
    codes, scale, z, x = w4_case(g, M, N, 128 * 34 + group, group, True)
    w, plain = ops.pack_w4(codes, scale, z, group), w4_weight(codes, scale, z, group)
    for norm in (False, True):
        for swiglu in (False, True):
            got = ops.gemv_w4(x, w, epilogue="swiglu" if swiglu else "bias", norm_eps=1e-6 if norm else None)
            near(got, *w4_reference(plain, scale, group, x, 1e-6 if norm else None, None, None, swiglu))


def test_gemv_w4_forms_of_the_call(ops):
    """one row as a vector, rows with a stride, the residual overwritten in place, another stream, rows that do not touch one another"""
    g = gen(3)
    codes, scale, z, x = w4_case(g, 6, 90, 384, 128, True)
    w = ops.pack_w4(codes, scale, z)
    full = ops.gemv_w4(x, w)
    assert torch.equal(ops.gemv_w4(x[2], w), full[2])
    wide = torch.zeros((6, 512), dtype=BF, device="cuda")
    wide[:, 64:448] = x
    assert torch.equal(ops.gemv_w4(wide[:, 64:448], w), full)
    assert torch.equal(ops.gemv_w4(x[::2], w), full[::2])
    r = randn(g, 6, 90).to(BF)
    want = ops.gemv_w4(x, w, res=r)
    got = ops.gemv_w4(x, w, res=r, out=r)
    assert got is r and torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.gemv_w4(x, w)
    side.synchronize()
    assert torch.equal(other, full)
    x2 = x.clone()
    x2[4] = float("nan")
    got = ops.gemv_w4(x2, w)
    assert got[4].isnan().all() and torch.equal(got[:4], full[:4]) and torch.equal(got[5], full[5])
    assert torch.equal(ops.gemv_w4(torch.zeros_like(x), w, norm_eps=1e-6), torch.zeros_like(full))


def test_gemv_w4_is_deterministic_and_replays(ops):
    g = gen(4)
    codes, scale, z, x = w4_case(g, 9, 700, 1024, 64, True)
    w = ops.pack_w4(codes, scale, z, 64)
    first = ops.gemv_w4(x, w, norm_eps=1e-6)
    assert all(torch.equal(ops.gemv_w4(x, w, norm_eps=1e-6), first) for _ in range(5))
    replays(lambda: ops.gemv_w4(x, w, norm_eps=1e-6), [x], [[randn(g, 9, 1024).to(BF)] for _ in range(4)], lambda a, b: check_equal(a, b))


def check_equal(a, b):
    assert torch.equal(a, b)


@pytest.mark.parametrize("group,zero_point", [(32, True), (64, False), (128, True), (128, False)])
def test_quantize_w4(ops, group, zero_point):
    """every weight within half a step of what it stands for (the scale is rounded to bf16, 2^-8, which the 15 steps of a group feel: 15 / 256 of a
    step more; a zero point is a whole number, another half step at the ends), and gemv_w4 of it is the product with those values"""
    g = gen(5)
    w = (randn(g, 70, 512) * 0.05 + 0.01).to(BF)
    w[3] = 0
    w[4, :128] = w[4, :128].abs()
    norm_w = (1 + 0.1 * randn(g, 512)).to(BF)
    for nw in (None, norm_w):
        q = ops.quantize_w4(w, group, zero_point, norm_w=nw)
        eye = torch.eye(512, device="cuda").to(BF)
        back = torch.cat([ops.gemv_w4(eye[i:i + 64], q) for i in range(0, 512, 64)]).T.to(F64)
        exact = w.to(F64) if nw is None else (w.float() * nw.float()).to(F64)
        parts = exact.view(70, -1, group)
        step = ((parts.amax(-1).clamp_min(0) - parts.amin(-1).clamp_max(0)) / 15 if zero_point else parts.abs().amax(-1) / 7)
        step = step.repeat_interleave(group, 1)
        assert ((back - exact).abs() <= step * (1.0 + 15 / 256) + HALF_BF * back.abs() + 1e-12).all()
        assert (back[3] == 0).all()


def test_gemv_w4_refusals(ops):
    g = gen(6)
    codes, scale, z, x = w4_case(g, 2, 40, 256, 128, True)
    w = ops.pack_w4(codes, scale, z)
    for bad in (lambda: ops.gemv_w4(x.float(), w), lambda: ops.gemv_w4(x[:, :128], w), lambda: ops.gemv_w4(x.T.contiguous().T, w),
                lambda: ops.gemv_w4(x, w, epilogue="gelu"), lambda: ops.gemv_w4(x, w, norm_eps=-1.0), lambda: ops.gemv_w4(x, w, bias=x[0]),
                lambda: ops.gemv_w4(x, w, res=x), lambda: ops.gemv_w4(x.cpu(), w), lambda: ops.pack_w4(codes, scale, z, 96),
                lambda: ops.pack_w4(codes, scale.float(), z), lambda: ops.pack_w4(codes, scale, z.int()), lambda: ops.pack_w4(codes, scale, z, 64),
                lambda: ops.quantize_w4(torch.zeros((8, 100), dtype=BF, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    from physicedit_amd._lib import PeError
    with pytest.raises(PeError, match="1 ... 64"):
        ops.gemv_w4(torch.zeros((65, 256), dtype=BF, device="cuda"), w)
    with pytest.raises(PeError, match="gated"):
        ops.gemv_w4(x, w, epilogue="swiglu")                       # 20 gate rows: no multiple of 16
    square = ops.pack_w4(torch.zeros((256, 128), dtype=torch.uint8, device="cuda"), torch.ones((256, 2), dtype=BF, device="cuda"))
    with pytest.raises(PeError, match="not x"):
        ops.gemv_w4(x, square, out=x)
    with pytest.raises(PeError, match="aligned"):
        ops.gemv_w4(torch.zeros((1, 264), dtype=BF, device="cuda")[:, 4:260], w)


# ---- the cache, written --------------------------------------------------------------------------------------------------------------------------

def quantise(x):
    """fp32 rows -> (e4m3 codes, fp32 scales), the definition"""
    top = x.abs().amax(-1)
    ok = top.isfinite()
    scale = torch.where(ok, (top * (1 / 448)).clamp_min(2.0 ** -126), torch.full_like(top, math.nan))
    return torch.where(ok[..., None], x / scale[..., None], torch.zeros_like(x)).to(F8), scale


def rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return x * cos + torch.cat([-b, a], -1) * sin


def bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype == F8 else t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)


def same(a, b):
    """equal bit for bit, any NaN for any NaN"""
    if a.dtype in (torch.float32, BF):
        assert torch.equal(a.isnan(), b.isnan())
        return torch.equal(bits(a.nan_to_num(0.0)), bits(b.nan_to_num(0.0)))
    return torch.equal(bits(a), bits(b))


def logical(cache):
    v = cache.v.reshape(cache.batch, cache.n_kv, cache.capacity, cache.head_dim)
    return dict(k=cache.k.clone(), v=v, k_scale=cache.k_scale.clone(), v_scale=cache.v_scale.clone())


def append_reference(old, k, v, start, q=None, cos=None, sin=None, positions=None):
    """plain loop over tokens: what the cache (as `logical` shows it) and q become"""
    new = {n: t.clone() for n, t in old.items()}
    B, T = k.shape[:2]
    cap = new["k"].shape[2]
    qo = None if q is None else torch.zeros(q.shape, dtype=BF, device="cuda")
    for b in range(B):
        for t in range(T):
            row = int(start[b]) + t
            if int(start[b]) < 0 or row >= cap:
                continue
            kk, vv = k[b, t].float(), v[b, t].float()
            if cos is not None:
                pos = row if positions is None else int(positions[b, t])
                c, s = ((x[pos].float() if 0 <= pos < x.shape[0] else torch.full_like(x[0].float(), math.nan)) for x in (cos, sin))
                kk = rotate(kk, c, s)
                if q is not None:
                    qo[b, t] = rotate(q[b, t].float(), c, s).to(BF)
            kq, ks = quantise(kk)
            vq, vs = quantise(vv)
            new["k"].view(torch.uint8)[b, :, row] = kq.view(torch.uint8)
            new["v"].view(torch.uint8)[b, :, row] = vq.view(torch.uint8)
            new["k_scale"][b, :, row], new["v_scale"][b, :, row] = ks, vs
    return new, qo


def check_append(ops, cache, k, v, start, **kw):
    old = logical(cache)
    q = ops.kv_append_e4m3(cache, k, v, start, **kw)
    want, wq = append_reference(old, k, v, start, **kw)
    got = logical(cache)
    for n in want:
        assert same(got[n], want[n]), n
    if wq is not None:
        assert same(q, wq)
    return q


def tables(rows, D, dtype):
    a = torch.arange(rows, device="cuda", dtype=F64)[:, None] * 1e4 ** (-torch.arange(0, D, 2, device="cuda", dtype=F64) / D)
    a = torch.cat([a, a], 1)
    return a.cos().to(dtype), a.sin().to(dtype)


@pytest.mark.parametrize("B,T,hq,hkv,D,cap,starts,dtype", [
    (1, 1, 28, 4, 128, 128, [77], BF),
    (1, 1, 2, 1, 64, 64, [63], torch.float32),
    (2, 3, 5, 1, 128, 192, [62, 0], torch.float32),
    (3, 64, 4, 2, 64, 192, [64, 1, 128], BF),
    (2, 130, 8, 8, 128, 256, [0, 127], BF),
    (4, 70, 6, 2, 128, 128, [-1, 100, 127, 128], BF),         # inactive, running over the end, the last row, full
    (1, 200, 3, 3, 64, 256, [33], torch.float32)])
def test_kv_append(ops, B, T, hq, hkv, D, cap, starts, dtype):
    g = gen(T)
    cache = ops.KVCacheE4M3(B, hkv, cap, D)
    cos, sin = tables(cap, D, dtype)
    everywhere = torch.zeros((B,), dtype=torch.int32, device="cuda")
    old = [randn(g, B, cap, hkv, D).to(BF) for _ in range(2)]
    check_append(ops, cache, *old, everywhere)                   # whole blocks; what stands there must survive the second write
    qkv = (3 * randn(g, B, T, hq + 2 * hkv, D)).to(BF)
    q, k, v = qkv.split([hq, hkv, hkv], 2)                       # strided views
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out = check_append(ops, cache, k, v, start, q=q, cos=cos, sin=sin)
    assert out.is_contiguous()
    check_append(ops, cache, k.transpose(1, 2).contiguous().transpose(1, 2), v.contiguous(), start)       # heads first, no rotation
    # a table row for each token, some of them outside the tables
    positions = torch.randint(-2, cap + 2, (B, T), generator=g, device="cuda").to(torch.int32)
    check_append(ops, cache, k, v, start, q=q, cos=cos, sin=sin, positions=positions)


def test_kv_append_odd_values(ops):
    """zeros, the smallest and largest numbers, infinities and NaN: a row that is not finite gets the scale NaN and codes of zero"""
    g = gen(8)
    D = 64
    k = randn(g, 1, 70, 1, D).to(BF)
    k[0, 0] = 0
    k[0, 1] *= 2.0 ** -130
    k[0, 2] = 1e-40
    k[0, 3] *= 1e37
    k[0, 4, 0, 5] = math.inf
    k[0, 5, 0, 63] = math.nan
    k[0, 6, 0, 1:] = 0
    cache = ops.KVCacheE4M3(1, 1, 128, D)
    check_append(ops, cache, k, k.clone(), torch.zeros((1,), dtype=torch.int32, device="cuda"))
    assert cache.k_scale[0, 0, 4].isnan() and cache.k_scale[0, 0, 5].isnan() and int(cache.k_scale.isnan().sum()) == 2
    assert not cache.k.float().isnan().any() and not cache.v.float().isnan().any()


def test_kv_append_replays(ops):
    """captured once, replayed with the row counter moved by the host: every replay writes where the counter says"""
    g = gen(9)
    B, T, hq, hkv, D, cap = 2, 2, 4, 2, 128, 128
    cos, sin = tables(cap, D, BF)
    a, b = ops.KVCacheE4M3(B, hkv, cap, D), ops.KVCacheE4M3(B, hkv, cap, D)
    q, k, v = (randn(g, B, T, h, D).to(BF) for h in (hq, hkv, hkv))
    start = torch.tensor([3, 61], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.kv_append_e4m3(a, k, v, start, q=q, cos=cos, sin=sin)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = ops.kv_append_e4m3(a, k, v, start, q=q, cos=cos, sin=sin)
    ops.kv_append_e4m3(b, k, v, start)
    ops.kv_append_e4m3(b, k, v, start, q=q, cos=cos, sin=sin)
    for _ in range(4):
        start += 5
        k.copy_(randn(g, B, T, hkv, D)), v.copy_(randn(g, B, T, hkv, D)), q.copy_(randn(g, B, T, hq, D))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.kv_append_e4m3(b, k, v, start, q=q, cos=cos, sin=sin)
        assert torch.equal(out, want)
        for n, t in logical(b).items():
            assert same(logical(a)[n], t), n


def test_kv_append_refusals(ops):
    cache = ops.KVCacheE4M3(2, 2, 64, 64)
    k = torch.zeros((2, 3, 2, 64), dtype=BF, device="cuda")
    s = torch.zeros((2,), dtype=torch.int32, device="cuda")
    cos, sin = tables(64, 64, BF)
    for bad in (lambda: ops.KVCacheE4M3(1, 1, 100, 64), lambda: ops.KVCacheE4M3(1, 1, 64, 96), lambda: ops.KVCacheE4M3(0, 1, 64, 64),
                lambda: ops.kv_append_e4m3(cache, k.float(), k, s), lambda: ops.kv_append_e4m3(cache, k[:1], k[:1], s),
                lambda: ops.kv_append_e4m3(cache, k, k[:, :2], s), lambda: ops.kv_append_e4m3(cache, k, k, s.long()),
                lambda: ops.kv_append_e4m3(cache, k, k, s[:1]), lambda: ops.kv_append_e4m3(cache, k, k, s, q=k),
                lambda: ops.kv_append_e4m3(cache, k, k, s, cos=cos), lambda: ops.kv_append_e4m3(cache, k, k, s, cos=cos, sin=sin.float()),
                lambda: ops.kv_append_e4m3(cache, k, k, s, cos=cos, sin=sin, positions=s), lambda: ops.kv_append_e4m3(cache, k.transpose(2, 3), k, s),
                lambda: ops.kv_append_e4m3(cache, torch.zeros((2, 3, 2, 68), dtype=BF, device="cuda")[..., 2:66], k, s)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


# ---- the cache, read back --------------------------------------------------------------------------------------------------------------------------

def attention_reference(q, cache, start, tree=None, scale=None):
    """-> result in 64 bits and how far fp32 may be from it: scores are sums of D products and three roundings more, p enters with its rounding to
    two bf16 (2^-16) and the exponential's (2^-21), sums of n terms; all relative to sum p |v| / sum p"""
    B, T, hq, D = q.shape
    l = logical(cache)
    k = l["k"].to(F64) * l["k_scale"].to(F64)[..., None]
    v = l["v"].to(F64) * l["v_scale"].to(F64)[..., None]
    cap, G = cache.capacity, hq // cache.n_kv
    scale = D ** -0.5 if scale is None else scale
    out, slack = torch.zeros((2, B, T, hq, D), dtype=F64, device="cuda")
    for b in range(B):
        s0 = min(int(start[b]), cap)
        n = 0 if s0 < 0 else min(s0 + T, cap)
        for t in range(T):
            word = (1 << (t + 1)) - 1 if tree is None else int(tree[b, t]) & (2 ** 64 - 1)
            see = [r for r in range(n) if r < s0 or (word >> (r - s0)) & 1]
            if not see:
                continue
            for h in range(hq):
                kk, vv = k[b, h // G, see], v[b, h // G, see]
                sc = kk @ q[b, t, h].to(F64) * scale
                off = (D + 4) * 2.0 ** -24 * ((kk.abs() @ q[b, t, h].to(F64).abs()) * scale)
                p = torch.softmax(sc, 0)
                out[b, t, h] = p @ vv
                slack[b, t, h] = (p * (2 * off.max() + 2.0 ** -15 + len(see) * 2.0 ** -24)) @ vv.abs()
    return out.view(B, T, -1), slack.view(B, T, -1)


def filled(ops, g, B, hkv, cap, D):
    cache = ops.KVCacheE4M3(B, hkv, cap, D)
    ops.kv_append_e4m3(cache, (1.2 * randn(g, B, cap, hkv, D)).to(BF), (randn(g, B, cap, hkv, D) + 0.2).to(BF), torch.zeros((B,), dtype=torch.int32, device="cuda"))
    return cache


@pytest.mark.parametrize("B,T,hq,hkv,D,cap,starts,mask", [
    (1, 1, 28, 4, 128, 128, [100], None),
    (1, 1, 28, 4, 128, 64, [0], None),                          # only itself
    (2, 1, 1, 1, 64, 64, [63, 62], None),
    (3, 1, 16, 8, 64, 1088, [1087, 500, 0], None),              # the cache's axis split over work-groups
    (6, 2, 14, 2, 128, 192, [0, 1, 63, 64, 65, 127], None),
    (2, 3, 20, 1, 64, 128, [-1, 40], None),                     # an inactive sequence; 60 rows a kv head
    (3, 5, 28, 4, 128, 320, [200, 0, 63], "tree"),
    (2, 21, 28, 4, 128, 192, [130, 7], "tree"),                 # 147 rows a kv head: several row blocks
    (2, 64, 4, 2, 64, 192, [64, 100], "tree"),
    (2, 64, 2, 2, 128, 128, [0, 64], "causal"),
    (3, 7, 5, 1, 128, 128, [64, 0, 126], "empty"),              # words of zero, contexts of none; running over the end
    (1, 9, 8, 4, 64, 128, [31], "every"),
    (2, 1, 7, 1, 128, 256, [256, 300], None)])                  # a full cache: the new token has no row
def test_kv_attention(ops, B, T, hq, hkv, D, cap, starts, mask):
    g = gen(cap + T)
    cache = filled(ops, g, B, hkv, cap, D)
    q = (1.5 * randn(g, B, hq, T, D)).to(BF).transpose(1, 2)     # strided
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    bit = torch.ones((), dtype=torch.int64, device="cuda") << torch.arange(T, device="cuda")
    tree = None
    if mask == "tree":                                          # token i descends from (i - 1) // 2
        up = torch.eye(T, dtype=F64)
        for i in range(1, T):
            up[i, (i - 1) // 2] = 1
        tree = (((torch.linalg.matrix_power(up, T) > 0).long() << torch.arange(T)).sum(1)).cuda().expand(B, T).contiguous()
    elif mask == "empty":
        tree = torch.where(torch.arange(T, device="cuda") % 2 == 0, torch.zeros_like(bit), bit).expand(B, T).contiguous()
    elif mask == "every":
        tree = torch.full((B, T), -1, dtype=torch.int64, device="cuda")
    got = ops.kv_attention_e4m3(q, cache, start, tree=tree)
    want, slack = attention_reference(q, cache, start, tree)
    assert got.shape == (B, T, hq * D) and got.dtype == BF
    near(got, want, slack)
    if mask == "empty":
        assert (got[1, 0::2] == 0).all()                        # no context and a word of zero
    if -1 in starts:
        assert (got[starts.index(-1)] == 0).all()
    if mask == "causal":
        bits_ = torch.stack([(1 << (t + 1)) - 1 if t < 63 else torch.tensor(-1) for t in torch.arange(T)]).cuda()
        assert torch.equal(ops.kv_attention_e4m3(q, cache, start, tree=bits_.long().expand(B, T).contiguous()), got)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 3, 5, 40])                       # 7, 21, 35, 280 rows a kv head: one, two, four row tiles, several blocks of them
def test_kv_attention_short_prefixes_in_a_long_cache(ops, T, D):
    """splits that have no rows write nothing, and what the workspace held before is not read into any result"""
    g = gen(D + T)
    B, hq, hkv, cap = 5, 14, 2, 8192
    cache = filled(ops, g, B, hkv, cap, D)
    q = (1.5 * randn(g, B, T, hq, D)).to(BF)
    start = torch.tensor([0, 100, 5000, -1, 64 * 20 - T], dtype=torch.int32, device="cuda")
    ws = ops.kv_attention_workspace(cache, T, hq)
    assert ws.numel() > 0
    got = [ops.kv_attention_e4m3(q, cache, start, workspace=ws.fill_(fill)) for fill in (255, 127, 0)]      # NaN, large numbers, zeros
    near(got[0], *attention_reference(q, cache, start))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and (got[0][3] == 0).all()


def test_kv_attention_masked_rows_do_not_leak(ops):
    """rows that are not finite, or anything at all behind the last token: no influence where masked, NaN where seen"""
    g = gen(12)
    B, T, hq, hkv, D, cap = 1, 4, 7, 1, 128, 256
    cache = filled(ops, g, B, hkv, cap, D)
    start = torch.tensor([90], dtype=torch.int32, device="cuda")
    k, v = randn(g, B, T, hkv, D).to(BF), randn(g, B, T, hkv, D).to(BF)
    q = randn(g, B, T, hq, D).to(BF)
    tree = torch.tensor([[1, 3, 5, 9]], dtype=torch.int64, device="cuda")       # three siblings below the first token
    ops.kv_append_e4m3(cache, k, v, start)
    clean = ops.kv_attention_e4m3(q, cache, start, tree=tree)
    for spoil in (math.nan, math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[0, 1, 0, 3], v2[0, 2, 0, 100] = spoil, spoil
        ops.kv_append_e4m3(cache, k2, v2, start)
        junk = torch.full((B, cap - 94, hkv, D), spoil, dtype=BF, device="cuda")
        ops.kv_append_e4m3(cache, junk, junk, start + 94)
        got = ops.kv_attention_e4m3(q, cache, start, tree=tree)
        assert torch.equal(got[0, 0], clean[0, 0]) and torch.equal(got[0, 3], clean[0, 3])
        assert got[0, 1].isnan().all() and got[0, 2].isnan().all()
    q2 = q.clone()
    q2[0, 3, 2] = math.nan
    ops.kv_append_e4m3(cache, k, v, start)
    got = ops.kv_attention_e4m3(q2, cache, start, tree=tree).view(T, hq, D)
    ok = torch.ones((T, hq), dtype=torch.bool, device="cuda")
    ok[3, 2] = False
    assert torch.equal(got[ok], clean.view(T, hq, D)[ok]) and got[3, 2].isnan().all()


def test_kv_attention_large_scores_and_scale(ops):
    """one score far above the rest, all scores far below zero, a scale of one's own"""
    g = gen(13)
    cache = ops.KVCacheE4M3(1, 1, 128, 64)
    k, v = randn(g, 1, 100, 1, 64).to(BF), randn(g, 1, 100, 1, 64).to(BF)
    k[0, 70] *= 40
    ops.kv_append_e4m3(cache, k, v, torch.zeros((1,), dtype=torch.int32, device="cuda"))
    start = torch.tensor([99], dtype=torch.int32, device="cuda")
    q = torch.cat([k[:, 70:71] * 3, -k[:, 70:71] * 3, randn(g, 1, 1, 1, 64).to(BF)], 2)
    for scale in (None, 1.0, 0.01, 0.0):
        got = ops.kv_attention_e4m3(q, cache, start, scale=scale)
        want, slack = attention_reference(q, cache, start, scale=scale)
        near(got, want, slack)


def test_kv_attention_streams_and_replays(ops):
    g = gen(14)
    B, T, hq, hkv, D, cap = 2, 3, 8, 2, 128, 1024
    cache = filled(ops, g, B, hkv, cap, D)
    start = torch.tensor([700, 20], dtype=torch.int32, device="cuda")
    q = randn(g, B, T, hq, D).to(BF)
    first = ops.kv_attention_e4m3(q, cache, start)
    assert all(torch.equal(ops.kv_attention_e4m3(q, cache, start), first) for _ in range(5))
    ws = ops.kv_attention_workspace(cache, T, hq)
    assert ws.numel() > 0 and torch.equal(ops.kv_attention_e4m3(q, cache, start, workspace=ws), first)
    streams = [torch.cuda.Stream() for _ in range(2)]            # two calls at once
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([ops.kv_attention_e4m3(q, cache, start) for _ in range(8)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for os_ in outs for o in os_)
    new = [[randn(g, B, T, hq, D).to(BF), torch.tensor(s, dtype=torch.int32, device="cuda")] for s in ([0, 1021], [63, 64], [-1, 512], [1000, 3])]
    replays(lambda: ops.kv_attention_e4m3(q, cache, start), [q, start], new, check_equal)


def test_kv_attention_past_32_bits(ops):
    """a cache whose bytes pass 2^32: the last sequence and the last head read their own rows"""
    g = gen(15)
    B, hkv, cap, D = 5, 4, 2 ** 21, 128                          # 5.4e9 bytes of keys
    cache = ops.KVCacheE4M3(B, hkv, cap, D)
    T = 90
    k, v = randn(g, B, T, hkv, D).to(BF), randn(g, B, T, hkv, D).to(BF)
    start = torch.tensor([0, 5, 9, 1, cap - T], dtype=torch.int32, device="cuda")
    ops.kv_append_e4m3(cache, k, v, start)
    small = ops.KVCacheE4M3(1, hkv, 128, D)
    zero = torch.zeros((1,), dtype=torch.int32, device="cuda")
    ops.kv_append_e4m3(small, k[4:], v[4:], zero)
    for n in ("k", "k_scale", "v_scale"):
        assert same(getattr(cache, n)[4, :, cap - T:], getattr(small, n)[0, :, :T]), n
    assert same(cache.v[4].reshape(hkv, -1, D)[:, cap - T:], small.v[0].reshape(hkv, -1, D)[:, :T])
    q = randn(g, B, 1, 8, D).to(BF)
    # only itself and the 89 rows before it are not zero: the rest have a score of 0 and a value of 0
    got = ops.kv_attention_e4m3(q, cache, start + T - 1)[4].float()
    kk, vv = (small.__dict__[n][0, :, :T].float() * small.__dict__[s][0, :, :T, None] for n, s in (("k", "k_scale"),) * 2)
    vv = small.v[0].reshape(hkv, 128, D)[:, :T].float() * small.v_scale[0, :, :T, None]
    sc = (q[4, 0].float().view(hkv, 2, D) @ kk.transpose(1, 2)).to(F64) / math.sqrt(D)
    w = sc.exp()
    want = ((w @ vv.to(F64)) / (w.sum(-1, keepdim=True) + (cap - T))).reshape(1, -1)
    # the rows of zeros add exp(0 - max) each, the same number 2^21 / (splits * 4 waves * 64 lanes) times in a row: fewer than 2^13 terms of one size, and
    # the sums of them, are off by less than 2^13 2^-24 = 2^-11 of the denominator; the numerator's 90 terms by 2^-15 (their two bf16) each
    assert ((got.to(F64) - want).abs() <= (HALF_BF + 2.0 ** -10) * want.abs() + 2.0 ** -14 * (w @ vv.to(F64).abs() / (w.sum(-1, keepdim=True) + (cap - T))).reshape(1, -1)).all()


def test_kv_attention_refusals(ops):
    cache = ops.KVCacheE4M3(2, 2, 64, 64)
    q = torch.zeros((2, 3, 4, 64), dtype=BF, device="cuda")
    s = torch.zeros((2,), dtype=torch.int32, device="cuda")
    t = torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    for bad in (lambda: ops.kv_attention_e4m3(q.float(), cache, s), lambda: ops.kv_attention_e4m3(q[:1], cache, s), lambda: ops.kv_attention_e4m3(q[:, :, :3], cache, s),
                lambda: ops.kv_attention_e4m3(q, cache, s.long()), lambda: ops.kv_attention_e4m3(q, cache, s, tree=t.int()),
                lambda: ops.kv_attention_e4m3(q, cache, s, tree=t[:, :2]), lambda: ops.kv_attention_e4m3(q, cache, s, out=q),
                lambda: ops.kv_attention_e4m3(torch.zeros((2, 65, 4, 64), dtype=BF, device="cuda"), cache, s), lambda: ops.kv_attention_e4m3(q.cpu(), cache, s)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    big = ops.KVCacheE4M3(1, 1, 1024, 64)
    from physicedit_amd._lib import PeError
    with pytest.raises(PeError, match="workspace"):
        ops.kv_attention_e4m3(q[:1], big, s[:1], workspace=torch.empty((16,), dtype=torch.uint8, device="cuda"))


# ---- next-token scores ----------------------------------------------------------------------------------------------------------------------------

def scores_reference(logits, counts=None, penalties=None, bias=None, allowed=None):
    x = logits.float().clone()
    R, V = x.shape
    if counts is not None:
        c = counts.int() & 0xffff
        made = (c & 0x7fff).float()
        p = torch.tensor([[1.0, 0, 0]], device="cuda") if penalties is None else penalties.view(-1, 3)
        rep, pres, freq = p[:, 0:1], p[:, 1:2], p[:, 2:3]
        x = torch.where(c != 0, torch.where(x > 0, x / rep, x * rep), x)
        x = x - freq * made
        x = x - pres * (made > 0)
    if bias is not None:
        x = x + bias
    if allowed is not None:
        v = torch.arange(V, device="cuda")
        x[(((allowed.view(-1, allowed.shape[-1])[:, v // 32] >> (v % 32).int()) & 1) == 0).expand(R, V)] = -math.inf
    return x


def first_best(x):
    x = x.masked_fill(x.isnan(), -math.inf)
    v = torch.arange(x.shape[1], device="cuda").expand_as(x)
    best = v.masked_fill(x != x.amax(1, keepdim=True), x.shape[1]).amin(1)
    return torch.where(x.amax(1) == -math.inf, torch.full_like(best, -1), best).int()


def scores_case(g, R, V, dtype):
    logits = (3 * randn(g, R, V)).to(dtype)
    counts = torch.where(torch.rand((R, V), generator=g, device="cuda") < 0.2, torch.randint(-2 ** 15, 2 ** 15, (R, V), generator=g, device="cuda"), 0).to(torch.int16)
    counts[:, ::7] = torch.where(counts[:, ::7] != 0, 3, 0).to(torch.int16)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (R, (V + 31) // 32), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    return logits, counts, torch.tensor([1.3, 0.4, 0.01], device="cuda") * (1 + 0.1 * torch.rand((R, 3), generator=g, device="cuda")), randn(g, R, V), allowed


@pytest.mark.parametrize("R,V", [(1, 1), (1, 7), (2, 8), (3, 33), (1, 2048), (2, 2049), (5, 4097), (3, 8192), (1, 8193), (2, 16385), (1, 152064), (9, 50001)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_process_and_select(ops, R, V, dtype):
    g = gen(V)
    logits, counts, pen, bias, allowed = scores_case(g, R, V, dtype)
    for kw in (dict(), dict(counts=counts), dict(counts=counts, penalties=pen), dict(counts=counts, penalties=pen[0].contiguous()), dict(bias=bias),
               dict(bias=bias[0].contiguous()), dict(allowed=allowed), dict(allowed=allowed[0].contiguous(), bias=bias),
               dict(counts=counts, penalties=pen, bias=bias, allowed=allowed)):
        want = scores_reference(logits, **kw)
        got = ops.process_logits(logits, **kw)
        assert got.dtype == torch.float32 and same(got, want), sorted(kw)
        assert torch.equal(ops.select_token(logits, **kw), first_best(want)), sorted(kw)


def test_select_ties_and_odd_values(ops):
    V = 5000
    x = torch.zeros((7, V), device="cuda")
    x[1, 4999] = x[1, 3000] = x[1, 2999] = 5
    x[2] = -math.inf
    x[3] = math.nan
    x[4], x[4, 17] = math.nan, -3
    x[5, 100], x[5, 4000] = math.inf, math.inf
    x[6], x[6, 4444] = -math.inf, -1e30
    want = torch.tensor([0, 2999, -1, -1, 17, 100, 4444], device="cuda", dtype=torch.int32)
    assert torch.equal(ops.select_token(x), want)
    none = torch.zeros((V + 31) // 32, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.select_token(x, allowed=none), torch.full_like(want, -1))
    assert (ops.process_logits(x, allowed=none) == -math.inf).all()          # NaN and infinities in masked places too
    one = none.clone()
    one[4321 // 32] = 1 << (4321 % 32)
    y = torch.where(torch.arange(V, device="cuda") == 4321, -1e38, math.nan).expand(2, V).contiguous()
    assert torch.equal(ops.select_token(y, allowed=one), torch.full((2,), 4321, dtype=torch.int32, device="cuda"))


def test_logits_with_a_row_stride(ops):
    g = gen(21)
    wide = randn(g, 4, 1003).to(BF)
    view = wide[:, 1:1000]                                       # rows at odd addresses
    assert torch.equal(ops.process_logits(view), view.float())
    assert torch.equal(ops.select_token(view), first_best(view.float()))
    assert torch.equal(ops.select_token(view[1:2]), first_best(view[1:2].float()))


def test_token_counts(ops):
    """ids given twice count twice, ids outside the vocabulary are padding, 32767 is the end, neighbours in a word stay as they are"""
    V = 1001
    counts = torch.zeros((3, V), dtype=torch.int16, device="cuda")
    ids = torch.randint(-3, V + 3, (3, 3000), generator=gen(22), device="cuda").to(torch.int32)
    ids[0, :700] = 500
    ops.token_counts_add(counts, ids)
    want = torch.zeros((3, V + 6), dtype=torch.int64, device="cuda").scatter_add_(1, ids.long() + 3, torch.ones_like(ids, dtype=torch.int64))[:, 3:V + 3]
    assert torch.equal(counts.long(), want)
    ops.token_counts_add(counts, ids[:, :50].contiguous(), prompt=True)
    seen = torch.zeros((3, V + 6), dtype=torch.bool, device="cuda").scatter_(1, ids[:, :50].long() + 3, True)[:, 3:V + 3]
    assert torch.equal(counts < 0, seen) and torch.equal(counts.long() & 0x7fff, want)
    counts[1, 7], counts[1, 8] = 32766, -1
    ops.token_counts_add(counts, torch.tensor([[-1] * 4, [7, 7, 7, 8], [-1] * 4], dtype=torch.int32, device="cuda"))
    assert int(counts[1, 7]) == 32767 and int(counts[1, 8]) == -1


def test_select_updates_the_decode_state(ops):
    """counts, token, list of tokens and step counter as the captured decode step keeps them: greedy with a repetition penalty, replayed"""
    g = gen(23)
    V, n = 3001, 12
    logits = (2 * randn(g, 1, V)).to(BF)
    pen = torch.tensor([2.0, 0.5, 0.25], device="cuda")
    counts, twin = torch.zeros((2, 1, V), dtype=torch.int16, device="cuda")
    token, out_ids, step = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")

    def one():
        ops.select_token(logits, counts=counts, penalties=pen, update_counts=True, out=token, out_ids=out_ids, step=step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    counts.zero_(), step.zero_(), out_ids.zero_()
    want = []
    for i in range(n + 2):                                       # two steps past the list: nothing is written there, the counter goes on
        best = int(first_best(scores_reference(logits, twin, pen)))
        want.append(best)
        twin[0, best] += 1
        graph.replay()
        torch.cuda.synchronize()
        assert int(token) == best and int(step) == i + 1 and torch.equal(counts, twin)
    assert out_ids.tolist() == want[:n] and len(set(want)) > 3


def test_logits_refusals(ops):
    x = torch.zeros((2, 40), device="cuda")
    c = torch.zeros((2, 40), dtype=torch.int16, device="cuda")
    t = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.process_logits(x.half()), lambda: ops.process_logits(x[0]), lambda: ops.process_logits(x.T), lambda: ops.process_logits(x[:, :0]),
                lambda: ops.process_logits(x, penalties=x[:, :3].contiguous()), lambda: ops.process_logits(x, counts=c[0]), lambda: ops.process_logits(x, counts=c.int()),
                lambda: ops.process_logits(x, bias=x[:, :39].contiguous()), lambda: ops.process_logits(x, allowed=t), lambda: ops.process_logits(x, allowed=c),
                lambda: ops.process_logits(x, counts=c, penalties=x[:, :2].contiguous()), lambda: ops.process_logits(x, out=c), lambda: ops.process_logits(x.cpu()),
                lambda: ops.select_token(x, update_counts=True), lambda: ops.select_token(x, step=t[0, :1].contiguous(), out_ids=t[0]),
                lambda: ops.select_token(x, out=t), lambda: ops.token_counts_add(c, t.long()), lambda: ops.token_counts_add(c, t[:1]),
                lambda: ops.token_counts_add(c[:, ::2], t), lambda: ops.token_counts_add(c.int(), t)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    from physicedit_amd._lib import PeError
    with pytest.raises(PeError, match="workspace"):
        ops.select_token(torch.zeros((2, 50000), device="cuda"), workspace=torch.empty((8,), dtype=torch.uint8, device="cuda"))


def test_results_over_their_inputs(ops):
    """exactly over an input where the documentation allows it; any other overlap is refused, whichever side begins first"""
    g = gen(12)
    codes, scale, z, _ = w4_case(g, 1, 96, 128, 64, True)
    w = ops.pack_w4(codes, scale, z, 64)
    flat = randn(g, 4096).to(BF)
    x, before = flat[1024:1024 + 256].view(2, 128), flat.clone()
    for lo in (1024 - 64, 1024 + 64, 1024 + 128):                      # out [2, 96] across x's start, inside it, across its end
        with pytest.raises(ValueError, match="overlaps x"):
            ops.gemv_w4(x, w, out=flat[lo:lo + 192].view(2, 96))
    with pytest.raises(ValueError, match="overlaps res"):
        ops.gemv_w4(x, w, res=flat[2048:2240].view(2, 96), out=flat[2049:2241].view(2, 96))
    with pytest.raises(ValueError, match="overlaps bias"):
        ops.gemv_w4(x, w, bias=flat[2048:2144], out=flat[2048:2240].view(2, 96))
    assert torch.equal(ops.gemv_w4(x, w, out=flat[1280:1472].view(2, 96)), ops.gemv_w4(x, w)) and torch.equal(flat[:1280], before[:1280]) and torch.equal(flat[1472:], before[1472:])

    cache, twin = ops.KVCacheE4M3(2, 2, 512, 64), ops.KVCacheE4M3(2, 2, 512, 64)
    start = torch.tensor([5, 300], dtype=torch.int32, device="cuda")
    cos, sin = tables(512, 64, BF)
    for T, hq in ((1, 6), (3, 6), (9, 6), (40, 2), (64, 10)):          # one, two, four row tiles of the attention and more
        q, k, v = randn(g, 2, T, hq, 64).to(BF), randn(g, 2, T, 2, 64).to(BF), randn(g, 2, T, 2, 64).to(BF)
        want = ops.kv_append_e4m3(twin, k, v, start, q=q, cos=cos, sin=sin)
        with pytest.raises(ValueError, match="overlaps k"):
            ops.kv_append_e4m3(cache, k, v, start, q=q[:, :, :2], cos=cos, sin=sin, out=k)
        got = ops.kv_append_e4m3(cache, k, v, start, q=q, cos=cos, sin=sin, out=q)
        assert got is q and torch.equal(q, want)
        small, zero = ops.KVCacheE4M3(2, 2, 64, 64), torch.zeros_like(start)
        ops.kv_append_e4m3(small, k, v, zero)
        for c, s in ((cache, start), (small, zero)):                   # a cache walked in parts and one of one block
            y = ops.kv_attention_e4m3(want, c, s)
            over = want.clone()
            assert torch.equal(ops.kv_attention_e4m3(over, c, s, out=over.view(2, T, -1)), y) and torch.equal(over.view(2, T, -1), y)
        with pytest.raises(ValueError, match="overlaps q"):
            ops.kv_attention_e4m3(want[:1].expand(2, T, hq, 64), cache, start, out=want.view(2, T, -1))

    x = randn(g, 3, 1000)
    counts, pen, bias, allowed = scores_case(g, 3, 1000, torch.float32)[1:]
    want = ops.process_logits(x, counts, pen, bias, allowed)
    over = x.clone()
    assert torch.equal(ops.process_logits(over, counts, pen, bias, allowed, out=over), want) and torch.equal(over, want)
    room = torch.zeros((3001,), device="cuda")
    with pytest.raises(ValueError, match="overlaps logits"):
        ops.process_logits(room[:3000].view(3, 1000), out=room[1:].view(3, 1000))
    with pytest.raises(ValueError, match="overlaps bias"):
        ops.process_logits(x, bias=room[:1000], out=room[:3000].view(3, 1000))
    ids = torch.zeros((8,), dtype=torch.int32, device="cuda")
    for out, out_ids, step in ((ids[:1], ids[:4], ids[5:6]), (ids[5:6], ids[:4], ids[5:6]), (ids[6:7], ids[:4], ids[3:4])):
        with pytest.raises(ValueError, match="overlaps"):
            ops.select_token(x[:1], out=out, out_ids=out_ids, step=step)


@pytest.mark.parametrize("V", [1, 2, 7, 33, 1000, 1001])
@pytest.mark.parametrize("R", [1, 3])
@pytest.mark.parametrize("lead", [0, 1])
@pytest.mark.parametrize("n", [1, 40, 2500])
def test_token_counts_where_rows_share_words(ops, V, R, lead, n):
    """rows that begin or end in the middle of a 32-bit word: ids counted exactly, also the first and the last of a row, up to 32767; what lies around stays"""
    g = gen(V * 100 + R * 10 + lead)
    buf = torch.full((lead + R * V + 3,), -21555, dtype=torch.int16, device="cuda")
    counts = buf[lead:lead + R * V].view(R, V)
    assert counts.data_ptr() % 4 == 2 * lead
    counts.zero_()
    counts[:, -1] = 32767 - 5
    want = counts.long() & 0xffff
    for prompt in (False, True, False):
        ids = torch.randint(-1, V + 1, (R, n), generator=g, device="cuda").to(torch.int32)
        ids[:, ::3] = torch.where(torch.rand((R, (n + 2) // 3), generator=g, device="cuda") < 0.5, 0, V - 1).to(torch.int32)
        assert ops.token_counts_add(counts, ids, prompt=prompt) is counts
        for r in range(R):
            here = ids[r][(ids[r] >= 0) & (ids[r] < V)].long()
            if prompt:
                want[r, here] |= 0x8000
            else:
                want[r] = (want[r] & 0x8000) | ((want[r] & 0x7fff) + torch.bincount(here, minlength=V)).clamp_max(0x7fff)
        assert torch.equal(counts.long() & 0xffff, want)
    assert (buf[:lead] == -21555).all() and (buf[lead + R * V:] == -21555).all()
    for token in (0, V - 1):                                     # the greedy choice counts there too
        logits = torch.zeros((R, V), device="cuda")
        logits[:, token] = 1
        assert (ops.select_token(logits, counts=counts, update_counts=True) == token).all()
        want[:, token] = (want[:, token] & 0x8000) | ((want[:, token] & 0x7fff) + 1).clamp_max(0x7fff)
    assert torch.equal(counts.long() & 0xffff, want)
    assert (buf[:lead] == -21555).all() and (buf[lead + R * V:] == -21555).all()


def test_token_counts_of_neighbours_at_once(ops):
    """two callers whose counts meet inside a 32-bit word, at the same time"""
    V, n = 501, 4000
    buf = torch.zeros((2 * V + 1,), dtype=torch.int16, device="cuda")
    ids = torch.randint(0, V, (1, n), generator=gen(77), device="cuda").to(torch.int32)
    ids[:, ::2], ids[:, 1::4] = 0, V - 1
    parts = [buf[:V].view(1, V), buf[V:2 * V].view(1, V)]
    torch.cuda.synchronize()
    for p in parts:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(4):
                ops.token_counts_add(p, ids)
    torch.cuda.synchronize()
    want = (4 * torch.bincount(ids[0].long(), minlength=V))
    assert all(torch.equal(p[0].long(), want) for p in parts) and int(buf[-1]) == 0


@pytest.mark.parametrize("B,H,T,cap", [(64, 32, 1, 512), (128, 16, 3, 512), (1, 1, 5, 128), (1, 2, 40, 192)], ids=["1row", "2rowtiles", "4rowtiles", "40tokens"])
@pytest.mark.parametrize("size", [1e37, 4e35, 1e-30])
def test_kv_attention_values_of_any_size(ops, B, H, T, cap, size):
    """scores that rise from block to block while the values are close to fp32's largest (as a sum: the documented limit) or far below one: the result is
    their mean.  Each wave walks at least two blocks here."""
    g = gen(T + cap)
    G, D = 7, 64
    cache = ops.KVCacheE4M3(B, H, cap, D)
    n = cap - T
    k, v = torch.zeros((2, B, cap, H, D), device="cuda")
    k[..., 0] = torch.arange(cap, device="cuda").view(1, cap, 1) // 64 * (5.4 / (cap // 64 - 1))            # 7.8 in powers of two, from first block to last
    v += (torch.rand((B, cap, H, D), generator=g, device="cuda") - 0.3) * (size if size < 1e36 else 1.0)
    if size > 1e36:                                                                                          # one value of that size
        v[:, n - 20, :, 3] = size
    ops.kv_append_e4m3(cache, k.to(BF), v.to(BF), torch.zeros((B,), dtype=torch.int32, device="cuda"))
    q = torch.zeros((B, T, H * G, D), device="cuda")
    q[..., 0] = 1 + 0.01 * torch.arange(H * G, device="cuda") / (H * G)
    q = q.to(BF)
    start = torch.full((B,), n, dtype=torch.int32, device="cuda")
    got = ops.kv_attention_e4m3(q, cache, start, scale=1.0)
    l = logical(cache)
    for b, h in ((0, 0), (B - 1, H - 1)):
        here = {x: t[b:b + 1, h:h + 1] for x, t in l.items()}
        kk, vv = here["k"].to(F64) * here["k_scale"].to(F64)[..., None], here["v"].to(F64) * here["v_scale"].to(F64)[..., None]
        for t in range(T):
            s = q[b, t, h * G:(h + 1) * G].to(F64) @ kk[0, 0, :n + t + 1].T
            p = torch.softmax(s, -1)
            want, most = p @ vv[0, 0, :n + t + 1], p @ vv[0, 0, :n + t + 1].abs()
            # as attention_reference: D products and four roundings of scores up to 5.5, p as two bf16, sums of n terms
            near(got[b, t].view(H, G, D)[h], want, most * (2 * (D + 4) * 2.0 ** -24 * 5.5 + 2.0 ** -15 + n * 2.0 ** -24))
    assert got.isfinite().all()


@pytest.mark.parametrize("M,N,K,group,swiglu", [(1, 300, 2048, 64, False), (1, 3584, 18944, 128, False), (5, 4099, 640, 128, False), (20, 1000, 1408, 64, True),
                                                (33, 8200, 384, 32, False), (64, 96, 4096, 32, True)])
@pytest.mark.parametrize("norm", [False, True])
def test_gemv_w4_range_of_inputs(ops, M, N, K, group, swiglu, norm):
    """inputs of the documented largest size, 2^100 (2^50 with the norm), and tiny ones; scales bring the products back to about one.  A row beyond the range
    touches no other."""
    if swiglu:
        N = N // 32 * 32
    g = gen(N + K)
    codes, scale, z, x = w4_case(g, M, N, K, group, True)
    size = 50 if norm else 100
    for e in (size, -size):
        xe = (x.clamp(-1, 1) * 2.0 ** e).to(BF)
        xe[:, ::5] = 2.0 ** e
        se = scale if norm else (scale.float() * 2.0 ** -e).to(BF)                # the normalised rows are of about one already
        w, plain = ops.pack_w4(codes, se, z, group), w4_weight(codes, se, z, group)
        kw = dict(epilogue="swiglu" if swiglu else "bias", norm_eps=2.0 ** -120 if norm else None)
        got = ops.gemv_w4(xe, w, **kw)
        near(got, *w4_reference(plain, se, group, xe, 2.0 ** -120 if norm else None, None, None, swiglu))
        if M > 1:
            for big in (3.3e38, math.inf, math.nan):
                x2 = xe.clone()
                x2[M // 2, K // 3] = big
                again = ops.gemv_w4(x2, w, **kw)
                ok = torch.arange(M, device="cuda") != M // 2
                assert torch.equal(again[ok], got[ok])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 300, 2048), (5, 4099, 640), (7, 3584, 18944), (20, 1000, 1408), (33, 8200, 384), (64, 96, 18944)])
def test_gemv_w4_to_the_last_bit(ops, group, M, N, K):
    """Inputs of 20 ... 57 whose weights are zero beside sixteenths whose weights are one: every sum that the kernel forms, (128 + code) x and x over a group,
    is a multiple of 2^-4 below 143 * 57 * 128 < 2^20, so nothing is rounded before the result: a term lost or taken twice anywhere shows."""
    g = gen(N + group)
    G = K // group
    z = torch.randint(1, 15, (N, G), generator=g, device="cuda")
    codes = z.repeat_interleave(group, 1)
    x = torch.randint(20, 58, (M, K), generator=g, device="cuda").float()
    at = torch.arange(G, device="cuda") * group + torch.randint(0, group, (G,), generator=g, device="cuda")      # one input of every group
    on = torch.rand((N, G), generator=g, device="cuda") < max(4.0 / G, 0.1)                                     # some of them count
    x[:, at] = torch.randint(-15, 16, (M, G), generator=g, device="cuda").float() / 16
    codes[:, at] += torch.where(on, torch.where(torch.rand((N, G), generator=g, device="cuda") < 0.5, 1, -1), 0)
    scale = 2.0 ** torch.randint(-3, 1, (N, 1), generator=g, device="cuda").float().expand(N, G)
    w = ops.pack_w4((codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8), scale.to(BF).contiguous(), z.to(torch.uint8), group)
    want = x.to(F64) @ ((codes - z.repeat_interleave(group, 1)).to(F64) * scale.to(F64).repeat_interleave(group, 1)).T
    assert torch.equal(ops.gemv_w4(x.to(BF), w), want.float().to(BF))


@pytest.mark.parametrize("M,N,K,group", [(1, 3584, 18944, 128), (7, 3584, 18944, 64), (24, 3584, 18944, 32), (64, 3584, 18944, 128), (33, 5001, 3424, 32), (1, 37888, 3584, 128)])
def test_gemv_w4_every_output(ops, M, N, K, group):
    """Each output within half a step of bf16 and what fp32 can lose on the way.  A group: group / 8 roundings of partial sums of at most 143 sum |x| (an
    instruction rounds four times in 32 terms or less), the same for sum x times 143, and two more; the groups' errors are independent and of no
    preferred sign, as are the roundings of their running sum, which stays within sqrt(G) times the largest term or so of the result: six times the root of the
    sum of squares covers all outputs."""
    g = gen(K + M)
    codes, scale, z, x = w4_case(g, M, N, K, group, True)
    got = ops.gemv_w4(x, ops.pack_w4(codes, scale, z, group)).to(F64)
    w = w4_weight(codes, scale, z, group)
    want = x.to(F64) @ w.T
    G, s = K // group, scale.to(F64)
    xa = x.to(F64).abs().view(M, G, group).sum(2)
    of_groups = ((xa * (2 * (group / 8) + 2) * 143 * 2.0 ** -24).square() @ s.square().T).sqrt()
    of_sums = (G + 16) ** 0.5 * 2.0 ** -24 * (want.abs() + (G * ((x.to(F64).square() @ w.square().T))).sqrt())
    loss = 6 * (of_groups + of_sums)
    assert ((got - want).abs() <= HALF_BF * (want.abs() + loss) + loss).all()
    assert float(loss.max() / want.std()) < 0.02                     # far below what one wrong term does


def test_flags_that_have_no_truth(ops):
    """a flag that cannot be read as true or false is its own error, and nothing is launched"""
    counts, both = torch.zeros((1, 40), dtype=torch.int16, device="cuda"), torch.ones(2)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.token_counts_add(counts, torch.tensor([[3, 4]], dtype=torch.int32, device="cuda"), prompt=both)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.select_token(torch.zeros((1, 40), device="cuda"), counts=counts, update_counts=both)
    assert not counts.any()


def test_what_a_call_writes_lies_apart_from_all_it_reads(ops):
    """the small inputs too (row counters, trees, positions, ids), and the workspace: every overlap is refused before a launch"""
    raw = torch.zeros((1 << 16,), dtype=torch.uint8, device="cuda")
    view = lambda lo, dtype, *shape: raw[lo:lo + math.prod(shape) * dtype.itemsize].view(dtype).view(shape)
    B, T, hq, hkv, D = 2, 3, 4, 2, 64
    cache = ops.KVCacheE4M3(B, hkv, 1024, D)
    cos, sin = tables(1024, D, BF)
    k, q, start = torch.zeros((B, T, hkv, D), dtype=BF, device="cuda"), torch.zeros((B, T, hq, D), dtype=BF, device="cuda"), torch.zeros((B,), dtype=torch.int32, device="cuda")
    out4, out3 = view(0, BF, B, T, hq, D), view(0, BF, B, T, hq * D)
    inside = 64
    positions, tree = view(inside, torch.int32, B, T), view(inside, torch.int64, B, T)
    ws = raw[:ops.kv_attention_workspace(cache, T, hq).numel()]
    assert ws.numel() > 0
    V, wide = 20000, torch.zeros((1, 20000), device="cuda")
    counts = torch.zeros((1, V), dtype=torch.int16, device="cuda")
    sel = raw[:16384]
    one = lambda at: view(at, torch.int32, 1)
    calls = {
        "out: overlaps start": [lambda: ops.kv_append_e4m3(cache, k, k, view(inside, torch.int32, B), q=q, cos=cos, sin=sin, out=out4),
                                lambda: ops.kv_attention_e4m3(q, cache, view(inside, torch.int32, B), out=out3)],
        "out: overlaps positions": [lambda: ops.kv_append_e4m3(cache, k, k, start, q=q, cos=cos, sin=sin, positions=positions, out=out4)],
        "out: overlaps tree": [lambda: ops.kv_attention_e4m3(q, cache, start, tree=tree, out=out3)],
        "workspace: overlaps out": [lambda: ops.kv_attention_e4m3(q, cache, start, out=out3, workspace=ws), lambda: ops.select_token(wide, out=one(8), workspace=sel)],
        "workspace: overlaps q": [lambda: ops.kv_attention_e4m3(view(0, BF, B, T, hq, D), cache, start, workspace=ws)],
        "workspace: overlaps start": [lambda: ops.kv_attention_e4m3(q, cache, view(inside, torch.int32, B), workspace=ws)],
        "workspace: overlaps tree": [lambda: ops.kv_attention_e4m3(q, cache, start, tree=tree, workspace=ws)],
        "workspace: overlaps logits": [lambda: ops.select_token(view(0, torch.float32, 1, 10000), workspace=sel)],
        "workspace: overlaps counts": [lambda: ops.select_token(view(32768, torch.float32, 1, 8192)[:, :8192], counts=view(0, torch.int16, 1, 8192), workspace=sel)],
        "workspace: overlaps allowed": [lambda: ops.select_token(wide, allowed=view(0, torch.int32, (V + 31) // 32), workspace=sel)],
        "workspace: overlaps step": [lambda: ops.select_token(wide, out_ids=torch.zeros(4, dtype=torch.int32, device="cuda"), step=one(8), workspace=sel)],
        "workspace: overlaps out_ids": [lambda: ops.select_token(wide, out_ids=one(12), step=torch.zeros(1, dtype=torch.int32, device="cuda"), workspace=sel)],
        "counts: overlaps tokens": [lambda: ops.token_counts_add(view(0, torch.int16, 1, 100), view(8, torch.int32, 1, 4))]}
    for text, fs in calls.items():
        for f in fs:
            with pytest.raises(ValueError, match=text):
                f()
    assert not raw.any() and not counts.any()
