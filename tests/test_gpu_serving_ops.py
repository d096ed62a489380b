"""The operators around a quantized linear when serving, against plain implementations in 64 bits: residual + RMS norm
+ 8-bit output, the rotation by positions of several axes, the adapters of many requests."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ck():
    import comfy_kitchen

    return comfy_kitchen


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=FP32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _half_step(dtype):
    """A rounding to the type is off by at most this, relative to the value; the second figure is the smallest step's half."""
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------ residual + RMS norm + 8 bits


def _norm_ref(h, weight, eps, dtype):
    """The definition in 64 bits, of the sum as stored."""
    v = h.double()
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.to(dtype).double()


def _check_norm(got, h, weight, eps, dtype):
    ref = _norm_ref(h, weight, eps, dtype)
    half, least = _half_step(dtype)
    # fp32: a thread's sum of at most 64 squares, 10 levels of a tree, the division, the root (2 units) and two products: under 2^-17
    err, tol = (got.double() - ref).abs(), ref.abs() * (half + 2.0 ** -17) + least + 1e-37
    assert bool((err <= tol).all()), f"worst {((err - tol).max()).item()} over the bound"


WIDTHS = [32, 96, 512, 4096, 5120, 8224, 20000, 65568]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (FP16, FP16), (FP32, FP32), (BF16, FP32), (FP16, FP32)])
def test_norm_mxfp8(ck, width, dtype, stream):
    g = _gen(width)
    for rows, use_weight, eps in ((1, True, 1e-6), (3, False, 1e-5), (130, True, 1e-6)):
        x, res = _randn(g, rows, width, dtype=dtype), _randn(g, rows, width, dtype=stream, scale=3.0)
        w = _randn(g, width, dtype=dtype) if use_weight else None
        q, s, h, y = ck.add_rmsnorm_quantize_mxfp8(x, res, w, eps, return_norm=True)
        assert torch.equal(_bytes(h), _bytes((x.float() + res.float()).to(stream)))
        assert y.dtype == dtype and h.dtype == stream and q.shape == (rows, width)
        _check_norm(y, h, w, eps, dtype)
        rq, rs = ck.quantize_mxfp8(y)
        assert torch.equal(_bytes(q), _bytes(rq)) and torch.equal(_bytes(s), _bytes(rs))
        again = ck.add_rmsnorm_quantize_mxfp8(x, res, w, eps)
        assert len(again) == 3 and torch.equal(_bytes(again[0]), _bytes(q)) and torch.equal(_bytes(again[1]), _bytes(s))


def test_norm_mxfp8_against_the_oracle(ck):
    from oracle import ck_oracle as orc

    g = _gen(1)
    x, res, w = _randn(g, 37, 416, dtype=BF16), _randn(g, 37, 416, dtype=BF16), _randn(g, 416, dtype=BF16)
    q, s, _, y = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True)
    rq, rs = orc.quantize_mxfp8(y.cpu())
    assert torch.equal(_bytes(q).cpu(), _bytes(rq)) and torch.equal(_bytes(s).cpu(), _bytes(rs))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_norm_mxfp8_scales_over_the_whole_range(ck, dtype):
    """Blocks from the smallest numbers of the type to the largest, with amax at, just below and just above 448 x 2^k, zeros, infinities and NaN:
    the codes and scales are those of the quantizer for the norm as stored."""
    low, high = {BF16: (-133, 127), FP32: (-149, 127), FP16: (-24, 15)}[dtype]
    mags = []
    for k in range(low, high + 1):
        for m in (1.0, 1.75, 1.75 * (1 - torch.finfo(dtype).eps), 1.75 * (1 + torch.finfo(dtype).eps)):
            mags.append(m * 2.0 ** k)
    mags = mags + [0.0, float("inf"), float("nan")]
    g = _gen(5)
    # x is +-1 and eps 0, so the norm is the weight with a sign: the weight is what is quantized
    width = 32 * len(mags)
    sign = torch.where(torch.rand(5, width, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    part = torch.rand(len(mags), 32, generator=g, device="cuda", dtype=torch.float64)
    part[torch.arange(len(mags)), torch.randint(0, 32, (len(mags),), generator=g, device="cuda")] = 1.0
    weight = (part * torch.tensor(mags, dtype=torch.float64, device="cuda")[:, None]).reshape(-1).to(dtype)
    q, s, h, y = ck.add_rmsnorm_quantize_mxfp8(sign.to(dtype), torch.zeros_like(sign).to(dtype), weight, 0.0, return_norm=True)
    expect_q, expect_s = ck.quantize_mxfp8(y, pad_32x=True)
    assert torch.equal(_bytes(q), _bytes(expect_q[:5])) and torch.equal(_bytes(s), _bytes(expect_s))
    finite = torch.isfinite(weight.float())
    assert torch.equal(y[:, finite].abs().double(), weight[finite].abs().double().expand(5, -1))


@pytest.mark.parametrize("width", [1, 7, 16, 100, 1315, 4096, 8192, 33000])
@pytest.mark.parametrize("dtype,stream,out", [(BF16, BF16, torch.float8_e4m3fn), (FP16, FP32, torch.float8_e5m2), (FP32, FP32, torch.float8_e4m3fn)])
def test_norm_fp8(ck, width, dtype, stream, out):
    g = _gen(width + 5)
    x, res, w = _randn(g, 5, 2, width, dtype=dtype), _randn(g, 5, 2, width, dtype=stream), _randn(g, width, dtype=dtype)
    scale = torch.tensor([0.013], device="cuda")
    q, h, y = ck.add_rmsnorm_quantize_fp8(x, res, w, scale, 1e-6, out, return_norm=True)
    assert q.shape == x.shape and q.dtype == out and torch.equal(_bytes(h), _bytes((x.float() + res.float()).to(stream)))
    _check_norm(y, h, w, 1e-6, dtype)
    assert torch.equal(_bytes(q), _bytes(ck.quantize_per_tensor_fp8(y, scale, out)))
    assert torch.equal(_bytes(ck.add_rmsnorm_quantize_fp8(x, res, w, scale, 1e-6, out)[0]), _bytes(q))


def test_norm_strides_alignment_and_in_place(ck):
    g = _gen(2)
    wide = _randn(g, 9, 3 * 512, dtype=BF16)
    res_wide = _randn(g, 9, 1025, dtype=BF16)
    w = _randn(g, 513, dtype=BF16)[1:]                                    # not 32-byte aligned
    for x, res in ((wide[:, 512:1024], res_wide[:, 1:513]), (wide[:, 3:515], res_wide[:, :512]), (wide[::2, :512], res_wide[1::2, 5:517].clone().repeat(2, 1)[:5])):
        a = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True)
        b = ck.add_rmsnorm_quantize_mxfp8(x.contiguous(), res.contiguous(), w.clone(), return_norm=True)
        _check_norm(a[3], a[2], w, 1e-6, BF16)
        assert torch.equal(a[2], b[2])
        _check_norm(b[3], b[2], w, 1e-6, BF16)
        own = res.contiguous().clone()
        c = ck.add_rmsnorm_quantize_mxfp8(x.contiguous(), own, w.clone(), return_norm=True, sum_out=own)
        assert c[2] is own and torch.equal(own, b[2])
        for u, v in zip(b, c):
            assert torch.equal(_bytes(u), _bytes(v))
    scalar = _randn(g, 65, dtype=FP32)
    own = scalar.clone()[1:].reshape(1, 64)                               # in place and unaligned
    q, h = ck.add_rmsnorm_quantize_fp8(own * 0 + 1, own, None, torch.ones(1, device="cuda"), sum_out=own)
    assert torch.equal(own, (scalar[1:] + 1).reshape(1, 64)) and h is own
    x3 = _randn(g, 3, 4, 64, dtype=FP16).transpose(0, 1)                  # no [rows, width] view
    q, s, h = ck.add_rmsnorm_quantize_mxfp8(x3, x3, None)
    assert h.shape == (4, 3, 64) and torch.equal(h, (x3.float() * 2).half().contiguous())


def test_norm_rows_do_not_touch_each_other(ck):
    g = _gen(3)
    x, res, w = _randn(g, 6, 160, dtype=BF16), _randn(g, 6, 160, dtype=BF16), _randn(g, 160, dtype=BF16)
    clean = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True)
    x[1], x[3, 7], res[4] = float("inf"), float("nan"), -x[4]
    q, s, h, y = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True)
    for r in (0, 2, 5):
        assert torch.equal(q[r].view(torch.uint8), clean[0][r].view(torch.uint8)) and torch.equal(y[r], clean[3][r])
    assert not bool(h[4].any()) and not bool(y[4].any()) and not bool(q[4].view(torch.uint8).any())     # a row of zeros
    rq, rs = ck.quantize_mxfp8(y)
    assert torch.equal(_bytes(q), _bytes(rq)) and torch.equal(_bytes(s), _bytes(rs))
    assert bool(y[3].isnan().all()) and bool(h[1].isinf().all())


def test_norm_of_nothing(ck):
    e = torch.empty(0, 64, device="cuda", dtype=BF16)
    q, s, h = ck.add_rmsnorm_quantize_mxfp8(e, e)
    assert q.shape == (0, 64) and s.shape == (0, 4) and h.shape == (0, 64)


# ------------------------------------------------------------------ rotation


def _rope_ref(x, positions, freqs, axes, split, tokens_dim, inverse=False):
    v = x.double()
    pos = positions.double()
    pos = pos[None] if pos.dim() == 2 else pos
    axis = torch.repeat_interleave(torch.arange(len(axes)), torch.tensor(axes) // 2).to(x.device)
    angle = (pos[..., axis] * freqs).unsqueeze(3 - tokens_dim)
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    p = sum(axes) // 2
    out, size = v.clone(), v.abs()
    ia, ib = (slice(0, p), slice(p, 2 * p)) if split else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    a, b = v[..., ia], v[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    bound = torch.zeros_like(v)
    bound[..., ia] = bound[..., ib] = size[..., ia] + size[..., ib]
    return out, bound


def _check_rope(got, ref, bound):
    half, least = _half_step(got.dtype)
    # the angle's rounding (pi 2^-24), sine and cosine (1 unit each) and two products and a sum in fp32: under 2^-20 of |a| + |b|
    err, tol = (got.double() - ref).abs(), ref.abs() * half + bound * 2.0 ** -20 + least
    assert bool((err <= tol).all()), f"worst {((err - tol).max()).item()} over the bound"


ROPES = [
    # B, N, Hq, Hk, D, axes, split, tokens_dim, positions of each batch entry
    (2, 37, 6, 2, 128, (16, 56, 56), False, 2, False),
    (1, 300, 4, 4, 128, (44, 42, 42), False, 1, True),
    (16, 1, 32, 8, 128, (32, 48, 48), True, 2, True),
    (3, 17, 5, 1, 80, (32, 32), True, 2, True),          # part of the head
    (2, 19, 3, 3, 64, (64,), False, 1, False),
    (1, 33, 2, 2, 96, (6, 10, 12, 20), False, 2, True),  # vectors that turn in part
    (2, 9, 2, 1, 40, (10, 14), True, 1, False),          # pairs no multiple of 8
    (1, 5, 1, 1, 6, (2,), False, 2, False),              # head no multiple of 8
    (2, 11, 2, 2, 72, (16,), True, 2, False),            # an odd number of vectors passes through
    (1, 2, 1, 1, 256, (2, 2, 2, 2, 2, 2, 2, 242), True, 2, False),
    (1, 4000, 1, 1, 128, (128,), False, 2, False),
]


@pytest.mark.parametrize("shape", ROPES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rope_axes(ck, shape, dtype):
    b, n, hq, hk, d, axes, split, tokens_dim, each = shape
    g = _gen(n + d)
    freqs = ck.rope_axes_freqs(axes)
    heads = lambda h: _randn(g, *((b, n, h, d) if tokens_dim == 1 else (b, h, n, d)), dtype=dtype)  # noqa: E731
    q, k = heads(hq), heads(hk)
    positions = torch.randint(-1000, 1 << 24, (b if each else 1, n, len(axes)), generator=g, device="cuda")
    for pos in (positions, positions.int(), positions.double() + 0.25, (positions % 4096).float() + 0.5, positions[0] if not each else positions):
        oq, ok = ck.apply_rope_axes(q, k, pos, freqs, axes, split, tokens_dim)
        _check_rope(oq, *_rope_ref(q, pos, freqs, axes, split, tokens_dim))
        _check_rope(ok, *_rope_ref(k, pos, freqs, axes, split, tokens_dim))
        assert torch.equal(ck.apply_rope_axes1(k, pos, freqs, axes, split, tokens_dim), ok)
    back = ck.apply_rope_axes1(q, positions, freqs, axes, split, tokens_dim, inverse=True)
    _check_rope(back, *_rope_ref(q, positions, freqs, axes, split, tokens_dim, inverse=True))


@pytest.mark.parametrize("tokens_dim", [1, 2])
@pytest.mark.parametrize("split", [False, True])
def test_rope_axes_strides(ck, tokens_dim, split):
    """q and k where a fused projection leaves them, without a copy; positions in another order."""
    g = _gen(4)
    b, n, h, d, axes = 2, 21, 3, 64, (16, 24, 24)
    qkv = _randn(g, b, n, 3 * h * d, dtype=BF16)
    views = [qkv[..., i * h * d:(i + 1) * h * d].view(b, n, h, d) for i in range(2)]
    if tokens_dim == 2:
        views = [v.transpose(1, 2) for v in views]
    pos = torch.randint(0, 5000, (3, n, b), generator=g, device="cuda").permute(2, 1, 0)
    freqs = ck.rope_axes_freqs(axes, 1e6)
    got = ck.apply_rope_axes(*views, pos, freqs, axes, split, tokens_dim)
    for o, v in zip(got, views):
        assert o.is_contiguous()
        _check_rope(o, *_rope_ref(v, pos, freqs, axes, split, tokens_dim))
    odd = _randn(g, b, h, n, 2 * d, dtype=FP16)[..., ::2]                 # no unit stride
    odd = odd if tokens_dim == 2 else odd.transpose(1, 2)
    _check_rope(ck.apply_rope_axes1(odd, pos, freqs, axes, split, tokens_dim), *_rope_ref(odd, pos, freqs, axes, split, tokens_dim))
    off = _randn(g, b * h * n * d + 1, dtype=FP16)[1:].view(b, h, n, d)   # not 16-byte aligned
    off = off if tokens_dim == 2 else off.transpose(1, 2)
    _check_rope(ck.apply_rope_axes1(off, pos, freqs, axes, split, tokens_dim), *_rope_ref(off, pos, freqs, axes, split, tokens_dim))


def test_rope_axes_equals_the_table(ck):
    """The same rotation as apply_rope with the matrices of an image model's grid."""
    from comfy_kitchen.dit_stack import DiTConfig, rope_freqs

    cfg = DiTConfig(txt_tokens=32, img_grid=(8, 12))
    g = _gen(5)
    q, k = _randn(g, 1, 3, cfg.tokens, 128, dtype=BF16), _randn(g, 1, 3, cfg.tokens, 128, dtype=BF16)
    ids = torch.zeros(cfg.tokens, 3, dtype=torch.int64, device="cuda")
    ids[32:, 1] = torch.arange(8, device="cuda").repeat_interleave(12)
    ids[32:, 2] = torch.arange(12, device="cuda").repeat(8)
    freqs = ck.rope_axes_freqs(cfg.axes_dim, cfg.theta)
    table = ck.apply_rope(q, k, rope_freqs(cfg, "cuda"))
    for o, t, x in zip(ck.apply_rope_axes(q, k, ids, freqs, cfg.axes_dim), table, (q, k)):
        ref, bound = _rope_ref(x, ids, freqs, cfg.axes_dim, False, 2)
        _check_rope(o, ref, bound)
        _check_rope(t, ref, bound)


def test_rope_axes_inverse_is_the_gradient(ck):
    g = _gen(6)
    axes, n = (8, 12, 12), 7
    pos = torch.randint(0, 900, (n, 3), generator=g, device="cuda")
    freqs = ck.rope_axes_freqs(axes)
    x = _randn(g, 1, 2, n, 32)
    grad = _randn(g, 1, 2, n, 32)
    v = x.double().requires_grad_()
    _rope_ref(v, pos, freqs, axes, True, 2)[0].backward(grad.double())
    inv = ck.apply_rope_axes1(grad, pos, freqs, axes, True, inverse=True)
    bound = _rope_ref(grad, pos, freqs, axes, True, 2)[1]
    _check_rope(inv, v.grad, bound)
    # differences of the rotation itself: it is linear, so a step of 1 is exact but for fp32 rounding
    for i in (0, 5, 20, 31):
        step = torch.zeros_like(x)
        step[0, 1, 3, i] = 1.0
        change = ck.apply_rope_axes1(x + step, pos, freqs, axes, True).double() - ck.apply_rope_axes1(x, pos, freqs, axes, True).double()
        assert abs((change * grad.double()).sum().item() - inv[0, 1, 3, i].item()) <= 64 * 8 * 2.0 ** -20


def test_rope_axes_of_nothing(ck):
    freqs = ck.rope_axes_freqs((8,))
    q, k = torch.empty(1, 2, 0, 8, device="cuda"), torch.empty(1, 1, 0, 8, device="cuda")
    oq, ok = ck.apply_rope_axes(q, k, torch.empty(0, 1, device="cuda"), freqs, (8,))
    assert oq.shape == q.shape and ok.shape == k.shape
    g = _gen(7)
    q, none = _randn(g, 1, 2, 3, 8), torch.empty(1, 0, 3, 8, device="cuda")
    pos = torch.arange(3, device="cuda")[:, None]
    oq, ok = ck.apply_rope_axes(q, none, pos, freqs, (8,))
    assert torch.equal(oq, ck.apply_rope_axes1(q, pos, freqs, (8,))) and ok.shape == none.shape
    ok, oq = ck.apply_rope_axes(none, q, pos, freqs, (8,))
    assert torch.equal(oq, ck.apply_rope_axes1(q, pos, freqs, (8,))) and ok.shape == none.shape


# ------------------------------------------------------------------ adapters


def _lora_ref(y, x, a, b, ids, scales):
    """(result, the sum of the products' absolute values) in 64 bits; rows without an adapter are y's."""
    out, size = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero()[:, 0]
        if rows.numel():
            f = 1.0 if scales is None else scales[i].double()
            xd, ad, bd = x[rows].double(), a[i].double(), b[i].double()
            out[rows] += f * ((xd @ ad.T) @ bd.T)
            size[rows] = abs(f) * ((xd.abs() @ ad.abs().T) @ bd.abs().T)
    return out, size


def _check_lora(got, y, x, a, b, ids, scales):
    ref, size = _lora_ref(y, x, a, b, ids, scales)
    half, least = _half_step(y.dtype)
    # fp32 sums of K, then R products: at most K + R units of 2^-23 of the products' absolute sum; the low-rank
    # vector as two 16-bit parts: 2^-16 of it at most
    err, tol = (got.double() - ref).abs(), ref.abs() * half * 1.01 + size * ((x.shape[1] + a.shape[1]) * 2.0 ** -23 + 2.0 ** -16) + least
    assert bool((err <= tol).all()), f"worst {((err - tol).max()).item()} over the bound"
    # a rounding is off by half a step at most, so the whole is, too; what comes before it adds next to nothing
    assert err.norm() <= 1.05 * half * ref.norm() + least * err.numel() ** 0.5
    none = (ids < 0) | (ids >= a.shape[0])
    assert torch.equal(_bytes(got[none]), _bytes(y[none]))


def _lora_case(rows, k, n, rank, adapters, dtype, seed, kind):
    g = _gen(seed)
    x, y = _randn(g, rows, k, dtype=dtype), _randn(g, rows, n, dtype=dtype)
    a, b = _randn(g, adapters, rank, k, dtype=dtype, scale=k ** -0.5), _randn(g, adapters, n, rank, dtype=dtype, scale=0.5 * rank ** -0.5)
    if kind == "mixed":          # any order, ids outside on both sides
        ids = torch.randint(-1, adapters + 1, (rows,), generator=g, device="cuda")
    elif kind == "runs":         # requests one behind the other
        ids = (torch.arange(rows, device="cuda") * (adapters + 1) // rows) - 1
    else:
        ids = torch.full((rows,), adapters - 1, device="cuda")
    return x, y, a, b, ids, 0.5 + torch.rand(adapters, generator=g, device="cuda")


LORAS = [
    (1, 8, 8, 8, 1, "one"), (1, 4096, 4096, 16, 8, "one"), (2, 72, 40, 24, 3, "mixed"), (7, 1000, 264, 40, 5, "mixed"), (16, 512, 1000, 32, 16, "mixed"),
    (31, 200, 136, 8, 2, "runs"), (33, 1024, 512, 64, 4, "mixed"), (64, 2048, 1032, 32, 20, "mixed"), (65, 264, 520, 128, 3, "runs"), (127, 320, 64, 16, 300, "mixed"),
    (128, 640, 256, 256, 2, "mixed"), (129, 1032, 392, 72, 7, "runs"), (300, 4096, 24, 64, 40, "mixed"), (511, 136, 2056, 16, 3, "runs"),
    (1000, 768, 776, 200, 6, "runs"), (2049, 256, 512, 64, 9, "runs"), (4100, 512, 1544, 32, 4, "runs"),
    (513, 64, 64, 256, 2, "mixed"), (600, 264, 136, 24, 40, "mixed"), (777, 1032, 520, 200, 9, "mixed"), (1025, 8, 8, 8, 3, "mixed"), (2000, 72, 4104, 48, 300, "mixed"),
    (400, 4096, 4096, 128, 3, "runs"), (40, 8192, 8192, 256, 5, "mixed"), (9473, 200, 136, 72, 9, "mixed"), (9728, 1032, 264, 128, 5, "runs"), (19200, 520, 72, 16, 3, "runs"),
]


@pytest.mark.parametrize("case", LORAS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_lora(ck, case, dtype):
    rows, k, n, rank, adapters, kind = case
    x, y, a, b, ids, scales = _lora_case(rows, k, n, rank, adapters, dtype, rows + k, kind)
    got = ck.lora_add(y, x, a, b, ids, scales)
    _check_lora(got, y, x, a, b, ids, scales)
    assert torch.equal(ck.lora_add(y, x, a, b, ids, scales), got)          # the same sums every time
    _check_lora(ck.lora_add(y, x, a, b, ids.int()), y, x, a, b, ids, None)
    own = y.clone()
    assert ck.lora_add(own, x, a, b, ids, scales, out=own) is own and torch.equal(own, got)


@pytest.mark.parametrize("rows,n,rank", [(3, 96, 16), (40, 96, 16), (700, 96, 16), (600, 4104, 256), (16500, 520, 128), (20000, 264, 64)])
def test_lora_nothing_to_add(ck, rows, n, rank):
    x, y, a, b, _, scales = _lora_case(rows, 512, n, rank, 4, BF16, 8, "one")
    for value in (-1, 4, -2 ** 31, 2 ** 31 - 1):
        ids = torch.full((rows,), value, device="cuda", dtype=torch.int32)
        assert torch.equal(_bytes(ck.lora_add(y, x, a, b, ids, scales)), _bytes(y))
    for value in (2 ** 32, -2 ** 63, 2 ** 63 - 1):
        ids = torch.full((rows,), value, device="cuda")
        assert torch.equal(_bytes(ck.lora_add(y, x, a, b, ids, scales)), _bytes(y))


@pytest.mark.parametrize("rows,rank", [(700, 64), (5000, 128), (17000, 24), (3000, 256)])
def test_lora_some_tiles_without_adapters(ck, rows, rank):
    """Whole tiles that are copied between tiles that are not, in place and not, again and again."""
    x, y, a, b, _, scales = _lora_case(rows, 264, 1032, rank, 4, BF16, rows, "one")
    ids = (torch.arange(rows, device="cuda") // 150 * 7) % 11 - 3
    first = ck.lora_add(y, x, a, b, ids, scales)
    _check_lora(first, y, x, a, b, ids, scales)
    for _ in range(20):
        own = y.clone()
        ck.lora_add(own, x, a, b, ids, scales, out=own)
        assert torch.equal(ck.lora_add(y, x, a, b, ids, scales), first) and torch.equal(own, first)
    from comfy_kitchen.backends import cuda

    assert cuda.lora_device_status() == 0


@pytest.mark.parametrize("rows", [5, 70, 900])
def test_lora_keeps_infinities_in_their_rows(ck, rows):
    x, y, a, b, ids, scales = _lora_case(rows, 264, 136, 24, 4, BF16, 9, "mixed")
    clean = ck.lora_add(y, x, a, b, ids, scales)
    bad = torch.arange(rows, device="cuda") % 3 == 1
    x[bad] = float("nan")
    x[bad & (torch.arange(rows, device="cuda") % 2 == 0)] = float("inf")
    unused = 2
    ids[ids == unused] = 0
    a[unused], b[unused] = float("nan"), float("inf")
    clean = torch.where((ids == 0)[:, None], ck.lora_add(y, torch.where(bad[:, None], torch.zeros_like(x), x), a, b, ids, scales), clean)
    got = ck.lora_add(y, x, a, b, ids, scales)
    none = (ids < 0) | (ids >= 4)
    assert torch.equal(_bytes(got[none]), _bytes(y[none]))
    assert torch.equal(got[~bad], clean[~bad])
    assert not bool(got[bad & ~none].isfinite().any())


def test_lora_large_low_rank_values(ck):
    """A first product beyond fp16's range is no infinity, and a tiny one does not vanish."""
    g = _gen(10)
    for scale, rows in ((300.0, 4), (300.0, 700), (2.0 ** -11, 4), (2.0 ** -11, 700)):
        x, a = _randn(g, rows, 512, dtype=FP16, scale=scale), _randn(g, 2, 16, 512, dtype=FP16, scale=min(scale, 20.0))
        b = _randn(g, 2, 64, 16, dtype=FP16, scale=2.0 ** -12 if scale > 1 else 30.0)
        y = _randn(g, rows, 64, dtype=FP16, scale=1.0 if scale > 1 else 2.0 ** -10)
        ids = torch.arange(rows, device="cuda") % 2
        assert scale < 1 or ((x.double() @ a[0].double().T).abs().max() > 65504)
        _check_lora(ck.lora_add(y, x, a, b, ids), y, x, a, b, ids, None)


@pytest.mark.parametrize("rows", [6, 48, 800])
def test_lora_strides_and_batches(ck, rows):
    g = _gen(11)
    k, n, rank = 256, 128, 16
    qkv, wide = _randn(g, rows, 3 * n, dtype=BF16), _randn(g, rows, k + 64, dtype=BF16)
    a, b = _randn(g, 3, rank, k, dtype=BF16, scale=0.06), _randn(g, 3, n, rank, dtype=BF16, scale=0.1)
    ids = torch.arange(rows, device="cuda") % 4
    kept = qkv.clone()
    x, y = wide[:, 64:], qkv[:, n:2 * n]
    ck.lora_add(y, x, a, b, ids, out=y)                                    # a slice of a fused projection, in place
    _check_lora(qkv[:, n:2 * n], kept[:, n:2 * n].contiguous(), x, a, b, ids, None)
    assert torch.equal(qkv[:, :n], kept[:, :n]) and torch.equal(qkv[:, 2 * n:], kept[:, 2 * n:])
    x1, y1 = _randn(g, rows * k + 1, dtype=BF16)[1:].view(rows, k), _randn(g, rows, 2 * n, dtype=BF16)[:, ::2]   # unaligned, no unit stride
    _check_lora(ck.lora_add(y1, x1, a, b, ids), y1, x1, a, b, ids, None)
    x3, y3 = _randn(g, 2, rows // 2, k, dtype=BF16), _randn(g, 2, rows // 2, n, dtype=BF16)
    each = torch.tensor([2, 0], device="cuda")                             # one adapter per batch entry
    flat = each.repeat_interleave(rows // 2)
    got = ck.lora_add(y3, x3, a, b, each)
    assert got.shape == y3.shape
    _check_lora(got.reshape(rows, n), y3.reshape(rows, n), x3.reshape(rows, k), a, b, flat, None)
    _check_lora(ck.lora_add(y3, x3, a, b, flat.view(2, -1)).reshape(rows, n), y3.reshape(rows, n), x3.reshape(rows, k), a, b, flat, None)
    one = torch.tensor(1, device="cuda")                                   # one for everything
    _check_lora(ck.lora_add(y3, x3, a, b, one).reshape(rows, n), y3.reshape(rows, n), x3.reshape(rows, k), a, b, torch.ones_like(flat), None)
    shared = x3[:1].expand(2, -1, -1)                                      # the same rows for two requests
    _check_lora(ck.lora_add(y3, shared, a, b, each).reshape(rows, n), y3.reshape(rows, n), shared.reshape(rows, k), a, b, flat, None)


@pytest.mark.parametrize("rows,k,n", [(1, 64, 312576), (1, 312576, 64), (2, 64, 160000)])
def test_lora_few_rows_of_many_columns(ck, rows, k, n):
    """So many columns that the tiled kernels take a single row."""
    x, y, a, b, ids, scales = _lora_case(rows, k, n, 256, 2, BF16, 77, "one")
    _check_lora(ck.lora_add(y, x, a, b, ids, scales), y, x, a, b, ids, scales)


def test_lora_of_nothing(ck):
    e = torch.empty(0, 64, device="cuda", dtype=BF16)
    a, b = torch.zeros(1, 8, 64, device="cuda", dtype=BF16), torch.zeros(1, 32, 8, device="cuda", dtype=BF16)
    assert ck.lora_add(torch.empty(0, 32, device="cuda", dtype=BF16), e, a, b, torch.empty(0, device="cuda", dtype=torch.int32)).shape == (0, 32)


def test_layers_with_adapters(ck):
    """The linear layers on quantized weights call it beside their projection."""
    from comfy_kitchen.linear import MXFP8Linear, NVFP4Linear

    g = _gen(12)
    k, n, rows = 256, 384, 70
    a, b, scales = _randn(g, 3, 16, k, dtype=BF16, scale=0.06), _randn(g, 3, n, 16, dtype=BF16, scale=0.1), 0.5 + torch.rand(3, device="cuda")
    w = _randn(g, n, k, dtype=BF16, scale=0.06)
    mx = MXFP8Linear.from_linear(torch.nn.Linear(k, n, bias=False, device="cuda", dtype=BF16).requires_grad_(False))
    ts = w.float().abs().max().reshape(1) / (6 * 448)
    q, sf = ck.quantize_nvfp4(w, ts)
    nv = NVFP4Linear(k, n, bias=False, device="cuda")
    nv.load_state_dict({"weight": q, "weight_scale": sf.view(torch.uint8), "weight_scale_2": ts}, strict=False)
    x = _randn(g, rows, k, dtype=BF16)
    ids = torch.arange(rows, device="cuda") % 4
    for layer in (mx, nv):
        base = layer(x)
        layer.set_adapters(a, b, scales)
        assert torch.equal(layer(x), base)
        got = layer(x, ids)
        assert torch.equal(got, ck.lora_add(base, x, a, b, ids, scales))
        _check_lora(got, base, x, a, b, ids, scales)
        layer.set_adapters(None)
        with pytest.raises(ValueError):
            layer(x, ids)
    mx.set_adapters(a, b)
    three = mx(x.view(2, rows // 2, k), torch.tensor([1, 2], device="cuda"))
    assert torch.equal(three.view(rows, n), ck.lora_add(mx(x), x, a, b, torch.tensor([1, 2], device="cuda").repeat_interleave(rows // 2)))


# ------------------------------------------------------------------ together, on other streams, in graphs


def _front_end(ck, x, res, nw, wq, ws, a, b, ids, scales, pos, freqs, axes, heads, dim):
    """A served layer's attention front end: residual + norm -> MXFP8, shared QKV projection, adapters, rotation."""
    q8, s8, h, y = ck.add_rmsnorm_quantize_mxfp8(x, res, nw, return_norm=True)
    qkv = ck.scaled_mm_mxfp8(q8, wq, s8, ws)
    ck.lora_add(qkv, y, a, b, ids, scales, out=qkv)
    q, k, v = qkv.view(1, -1, 3, heads, dim).unbind(2)
    oq, ok = ck.apply_rope_axes(q, k, pos, freqs, axes, tokens_dim=1)
    return h, qkv, oq, ok, v


def _front_case(ck, rows, seed):
    g = _gen(seed)
    heads, dim, width, axes = 2, 64, 256, (16, 24, 24)
    w = _randn(g, 3 * heads * dim, width, dtype=BF16, scale=width ** -0.5)
    wq, ws = ck.quantize_mxfp8(w)
    a, b = _randn(g, 3, 16, width, dtype=BF16, scale=width ** -0.5), _randn(g, 3, 3 * heads * dim, 16, dtype=BF16, scale=0.1)
    pos = torch.randint(0, 4096, (rows, 3), generator=g, device="cuda")
    return [_randn(g, rows, width, dtype=BF16), _randn(g, rows, width, dtype=FP32), _randn(g, width, dtype=BF16), wq, ws, a, b,
            torch.arange(rows, device="cuda") % 4, 0.5 + torch.rand(3, generator=g, device="cuda"), pos, ck.rope_axes_freqs(axes), axes, heads, dim]


@pytest.mark.parametrize("rows", [1, 50, 700])
def test_layer_front_end(ck, rows):
    args = _front_case(ck, rows, rows)
    x, res, nw, wq, ws, a, b, ids, scales, pos, freqs, axes, heads, dim = args
    h, qkv, oq, ok, v = _front_end(ck, *args)
    q8, s8, h2, y = ck.add_rmsnorm_quantize_mxfp8(x, res, nw, return_norm=True)
    act, weight = ck.dequantize_mxfp8(q8, s8, FP32).double(), ck.dequantize_mxfp8(wq, ws, FP32).double()
    base = act @ weight.T
    ref, size = _lora_ref(base, y, a, b, ids, scales)
    # the projection's output and the sum are each rounded to bf16; 256 products in fp32 before that
    tol = 2.0 ** -8 * (base.abs() + ref.abs()) * 1.01 + (act.abs() @ weight.abs().T + size) * (300 * 2.0 ** -23 + 2.0 ** -16)
    assert bool(((qkv.double() - ref).abs() <= tol).all())
    parts = qkv.view(1, rows, 3, heads, dim).unbind(2)
    for o, p in ((oq, parts[0]), (ok, parts[1])):
        _check_rope(o, *_rope_ref(p, pos, freqs, axes, False, 1))
    assert torch.equal(h, h2) and torch.equal(v, parts[2])


@pytest.mark.parametrize("rows", [4, 700])
def test_front_end_on_another_stream_and_in_graphs(ck, rows):
    args, other = _front_case(ck, rows, 20), _front_case(ck, rows, 21)
    want, want_other = _front_end(ck, *args), _front_end(ck, *other)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _front_end(ck, *args)
    side.synchronize()
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for s in (args, other):      # two graphs in one memory pool: their workspaces lie in the same places
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=side):
            outs.append([t.clone() for t in _front_end(ck, *s)])
        graphs.append(graph)
    graphs[0].replay()
    first = [t.clone() for t in outs[0]]
    graphs[1].replay()
    for u, v in zip(first, want):
        assert torch.equal(u, v)
    for u, v in zip(outs[1], want_other):
        assert torch.equal(u, v)
    for i in (0, 1, 5, 7, 9):    # new inputs in the old places
        args[i].copy_(other[i])
    args[3].view(torch.uint8).copy_(other[3].view(torch.uint8))
    args[4].view(torch.uint8).copy_(other[4].view(torch.uint8))
    for i in (2, 6, 8):
        args[i].copy_(other[i])
    graphs[0].replay()
    for u, v in zip(outs[0], want_other):
        assert torch.equal(u, v)


def test_compiled_and_fake(ck):
    args = _front_case(ck, 9, 22)
    x, res, nw, a, b, ids, scales, pos, freqs, axes = args[0], args[1], args[2], args[5], args[6], args[7], args[8], args[9], args[10], args[11]
    y = torch.zeros(9, 384, device="cuda", dtype=BF16)
    torch.library.opcheck(torch.ops.comfy_kitchen.add_rmsnorm_quantize_mxfp8, (x, res, nw, 1e-6, True), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.comfy_kitchen.add_rmsnorm_quantize_fp8, (x, res, nw, scales[:1], 1e-6, 5, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.comfy_kitchen.lora_add, (y, x, a, b, ids, scales), test_utils=("test_schema", "test_faketensor"))
    q = torch.zeros(1, 9, 2, 64, device="cuda", dtype=BF16)
    torch.library.opcheck(torch.ops.comfy_kitchen.apply_rope_axes, (q, q, pos, freqs, list(axes), False, 1, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.comfy_kitchen.apply_rope_axes1, (q, pos, freqs, list(axes), False, 1, False), test_utils=("test_schema", "test_faketensor"))
