"""What the serving operators promise beyond their results on whole, separate, finite tensors."""
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


def _randn(g, *shape, dtype=BF16, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def _layers(ck, k, n, bias):
    """An NVFP4Linear and an MXFP8Linear of the same weight, with a bias that wants a gradient (as it does by default)."""
    from comfy_kitchen.linear import MXFP8Linear, NVFP4Linear

    g = _gen(12)
    plain = torch.nn.Linear(k, n, bias=bias, device="cuda", dtype=BF16)
    plain.weight.data.copy_(_randn(g, n, k, scale=k ** -0.5))
    ts = plain.weight.data.float().abs().max().reshape(1) / (6 * 448)
    q, sf = ck.quantize_nvfp4(plain.weight.data, ts)
    state = {"weight": q, "weight_scale": sf.view(torch.uint8), "weight_scale_2": ts}
    if bias:
        plain.bias.data.copy_(_randn(g, n))
        state["bias"] = plain.bias.data
    nv = NVFP4Linear(k, n, bias=bias, device="cuda")
    nv.load_state_dict(state, strict=False)
    return nv, MXFP8Linear.from_linear(plain)


def test_layers_with_a_bias_take_adapters(ck):
    k, n, rows = 256, 384, 70
    g = _gen(1)
    a, b = _randn(g, 3, 16, k, scale=0.06), _randn(g, 3, n, 16, scale=0.1)
    x, ids = _randn(g, rows, k), torch.arange(rows, device="cuda") % 4
    for layer in _layers(ck, k, n, True):
        layer.set_adapters(a, b)
        base = layer(x)
        got = layer(x, ids)
        assert got.requires_grad == base.requires_grad
        assert torch.equal(got.detach(), ck.lora_add(base.detach(), x, a, b, ids))
        if got.requires_grad:
            grad = _randn(g, rows, n)
            want, = torch.autograd.grad(base, layer.bias, grad)
            have, = torch.autograd.grad(got, layer.bias, grad)
            assert torch.equal(have, want)
        with torch.no_grad():
            assert torch.equal(layer(x, ids), got.detach())


# ------------------------------------------------------------------ per-tensor FP8: infinities and NaN


def _fp8_ref(x, scale, out):
    """The definition on the CPU: a product rounded to x's type, clamped (NaN stays), rounded to 8 bits."""
    x, most = x.cpu(), torch.finfo(out).max
    inverse = (1.0 / scale.cpu()).to(x.dtype)
    return (x.float() * inverse.float()).to(x.dtype).float().clamp(-most, most).to(out)


def _same_codes(got, want):
    got, want = got.cpu(), want.cpu()
    nan = want.float().isnan()
    assert torch.equal(got.float().isnan(), nan)
    assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [1.0, 0.37, 1e-30, float("nan"), float("inf"), 0.0])
def test_fp8_quantizer_on_every_number_of_a_type(ck, dtype, out, scale):
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    scale = torch.tensor([scale], device="cuda")
    _same_codes(ck.quantize_per_tensor_fp8(x, scale, out), _fp8_ref(x, scale, out))
    odd = x[1:4099]                                                        # not aligned, no whole chunks
    _same_codes(ck.quantize_per_tensor_fp8(odd, scale, out), _fp8_ref(odd, scale, out))


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("dtype,stream,width", [(BF16, BF16, 4096), (FP16, FP32, 96), (FP32, FP32, 33), (BF16, FP32, 20000)])
def test_norm_fp8_keeps_infinities_and_nan(ck, dtype, stream, width, out):
    g = _gen(width)
    x, res, w = _randn(g, 6, width, dtype=dtype), _randn(g, 6, width, dtype=stream), _randn(g, width, dtype=dtype)
    x[1, 3], x[2], x[4, 0], x[4, 1] = float("nan"), float("inf"), float("inf"), -float("inf")
    for scale in (0.013, 1e-4):                                            # (the second one saturates)
        scale = torch.tensor([scale], device="cuda")
        q, h, y = ck.add_rmsnorm_quantize_fp8(x, res, w, scale, 1e-6, out, return_norm=True)
        assert bool(y[1].isnan().all()) and bool(q[1].float().isnan().all())
        _same_codes(q, _fp8_ref(y, scale, out))
        _same_codes(q, ck.quantize_per_tensor_fp8(y, scale, out))


# ------------------------------------------------------------------ outputs beside and over inputs


@pytest.mark.parametrize("rows", [3, 64, 700])
def test_lora_out_beside_its_inputs(ck, rows):
    g = _gen(rows)
    n = k = 128
    a, b, ids = _randn(g, 3, 16, k, scale=0.06), _randn(g, 3, n, 16, scale=0.1), torch.arange(rows, device="cuda") % 4
    buf = _randn(g, rows, 3 * n)
    y, x, kept = buf[:, :n], buf[:, n:2 * n], buf.clone()
    want = ck.lora_add(y.clone(), x.clone(), a, b, ids)
    ck.lora_add(y, x, a, b, ids, out=buf[:, 2 * n:])                       # a third column block of one buffer
    assert torch.equal(buf[:, 2 * n:], want) and torch.equal(buf[:, :2 * n], kept[:, :2 * n])
    ck.lora_add(y, x, a, b, ids, out=y)                                    # y's own
    assert torch.equal(y, want) and torch.equal(x, kept[:, n:2 * n])
    one = x.clone()                                                        # x, y and out in one place: h + B A h
    want_one = ck.lora_add(one, one, a, b, ids)
    ck.lora_add(one, one, a, b, ids, out=one)
    assert torch.equal(one, want_one)
    of_x = x.clone()                                                       # x's place
    ck.lora_add(kept[:, :n], of_x, a, b, ids, out=of_x)
    assert torch.equal(of_x, want)
    wide = _randn(g, rows, n + 64)                                         # out's row over part of x's
    x_part = wide[:, 64:].clone()
    ck.lora_add(kept[:, :n], wide[:, 64:], a, b, ids, out=wide[:, :n])
    assert torch.equal(wide[:, :n], ck.lora_add(kept[:, :n], x_part, a, b, ids))
    every = _randn(g, 3 * rows, n)
    every[0::3], every[1::3] = kept[:, :n], kept[:, n:2 * n]
    ck.lora_add(every[0::3], every[1::3], a, b, ids, out=every[2::3])      # every third row
    assert torch.equal(every[2::3], want) and torch.equal(every[0::3], kept[:, :n])
    rest = _randn(g, rows + 1, n)
    for yy, xx, out in ((rest[:-1], x, rest[1:]), (rest[1:], x, rest[:-1]), (kept[:, :n], rest[1:], rest[:-1]),
                        (buf[:, :n], x, buf[:, 64:n + 64])):
        before = out.clone()
        with pytest.raises(RuntimeError, match="overlaps"):
            ck.lora_add(yy, xx, a, b, ids, out=out)
        assert torch.equal(out, before)


@pytest.mark.parametrize("width,dtype,stream", [(4096, BF16, BF16), (96, FP16, FP16), (32, FP32, FP32), (20000, FP32, FP32), (40000, BF16, BF16)])
def test_norm_sum_over_its_inputs(ck, width, dtype, stream):
    g = _gen(width)
    x, res, w = _randn(g, 5, width, dtype=dtype), _randn(g, 5, width, dtype=stream), _randn(g, width, dtype=dtype)
    want = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True)
    for which in range(2):
        args = [x.clone(), res.clone()]
        got = ck.add_rmsnorm_quantize_mxfp8(*args, w, return_norm=True, sum_out=args[which])
        assert got[2] is args[which] and torch.equal(args[1 - which], (x, res)[1 - which])
        for u, v in zip(got, want):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
    both = x.to(stream)
    twice = ck.add_rmsnorm_quantize_mxfp8(both.to(dtype), both, w)[2]
    same = both.to(dtype)
    assert torch.equal(ck.add_rmsnorm_quantize_mxfp8(same, same, w, sum_out=same)[2], twice)   # (x, residual and h in one place)
    long = _randn(g, 6, width, dtype=stream)
    before = long.clone()
    for r, s in ((long[:5], long[1:]), (long[1:], long[:5])):
        with pytest.raises(RuntimeError, match="overlaps"):
            ck.add_rmsnorm_quantize_mxfp8(x, r, w, sum_out=s)
        with pytest.raises(RuntimeError, match="overlaps"):
            ck.add_rmsnorm_quantize_fp8(r, x.to(stream), w, torch.ones(1, device="cuda"), sum_out=s)
    assert torch.equal(long, before)


# ------------------------------------------------------------------ compiled, in place


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_in_place_forms_compiled(ck, backend):
    g = _gen(5)
    rows, width, n = 50, 256, 384
    x, res, w, scale = _randn(g, rows, width), _randn(g, rows, width, dtype=FP32), _randn(g, width), torch.tensor([0.02], device="cuda")
    a, b, ids = _randn(g, 3, 16, width, scale=0.06), _randn(g, 3, n, 16, scale=0.1), torch.arange(rows, device="cuda") % 4
    y = _randn(g, rows, n)

    def step(x, res, y, into):
        q, s, h, norm = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True, sum_out=res)     # the stream's own place
        q2, h2, norm2 = ck.add_rmsnorm_quantize_fp8(x, h, w, scale, return_norm=True, sum_out=into)
        ck.lora_add(y, norm, a, b, ids, out=y)                                                       # the projection's
        z = ck.lora_add(y, norm2, a, b, ids, out=torch.empty_like(y))
        return [q, s, q2, h + 1, h2 * 2, norm, norm2, z]

    def given():
        return [x.clone(), res.clone(), y.clone(), torch.zeros_like(res)]

    ours, theirs = given(), given()
    with torch.no_grad():
        want = step(*ours)
        got = torch.compile(step, fullgraph=True, backend=backend)(*theirs)
    for u, v in zip(want + ours, got + theirs):
        assert u.dtype == v.dtype and torch.equal(u.view(torch.uint8), v.view(torch.uint8))


def test_in_place_ops(ck):
    g = _gen(6)
    x, res, w = _randn(g, 9, 64), _randn(g, 9, 64), _randn(g, 64)
    a, b, ids, scale = _randn(g, 3, 16, 64), _randn(g, 3, 96, 16), torch.arange(9, device="cuda") % 4, torch.ones(1, device="cuda")
    y = _randn(g, 9, 96)
    ops, which = torch.ops.comfy_kitchen, ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.lora_add_out, (y, x, a, b, ids, None, torch.empty_like(y)), test_utils=which)
    for keep in (True, False):
        torch.library.opcheck(ops.add_rmsnorm_quantize_mxfp8_out, (x, res, w, 1e-6, keep, torch.empty_like(res)), test_utils=which)
        torch.library.opcheck(ops.add_rmsnorm_quantize_fp8_out, (x, res, w, scale, 1e-6, 5, keep, torch.empty_like(res)), test_utils=which)


# ------------------------------------------------------------------ adapters: workspaces


@pytest.mark.parametrize("rows", [700, 5000])
def test_lora_nothing_to_add_in_place_then_another(ck, rows):
    """In place and with no adapter asked for no CTA of the last kernel has work; what follows, in the same memory, must find the kernels
    before it done.  (A padded step of a captured graph.)"""
    g = _gen(rows)
    k, n, rank = 512, 1032, 64
    a, b = _randn(g, 4, rank, k, scale=0.05), _randn(g, 4, n, rank, scale=0.1)
    x, y = _randn(g, rows, k), _randn(g, rows, n)
    none, some = torch.full((rows,), -1, device="cuda"), torch.arange(rows, device="cuda") // 100 % 5
    want = ck.lora_add(y, x, a, b, some)
    own = y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(4):
            ck.lora_add(own, x, a, b, none, out=own)
            garbage = torch.full((1 << 22,), 0x7F7F7F7F, dtype=torch.int32, device="cuda")    # into the workspace that was given back
            del garbage
            got = ck.lora_add(own, x, a, b, some)
    for _ in range(50):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(own, y) and torch.equal(got, want)
    from comfy_kitchen.backends import cuda

    assert cuda.lora_device_status() == 0


@pytest.mark.parametrize("rows,k,n,rank", [(700, 512, 264, 64), (520, 264, 1032, 200), (5000, 1032, 520, 24), (17000, 256, 136, 128)])
def test_lora_workspace_needs_no_value(ck, rows, k, n, rank):
    """Through the C entry: whatever lies in the scratch, nothing behind its end is touched, and it is the call's own again the next time."""
    from comfy_kitchen import _native

    g = _gen(rows + n)
    a, b, scales = _randn(g, 5, rank, k, scale=k ** -0.5), _randn(g, 5, n, rank, scale=0.1), 0.5 + torch.rand(5, generator=g, device="cuda")
    x, y = _randn(g, rows, k), _randn(g, rows, n)
    ids = (torch.arange(rows, device="cuda") // 150 * 7) % 9 - 2           # tiles of several adapters, of one, of none
    want = ck.lora_add(y, x, a, b, ids, scales)
    need = _native.load().ck_lora_workspace_bytes(rows, k, n, rank)
    assert need > 0
    work, tail = torch.empty(need + 4096, dtype=torch.uint8, device="cuda"), 0x5A
    for fill in (0x00, 0xFF, 0x7F, 0x80, "random", "last"):
        if fill == "random":
            work.copy_(torch.randint(0, 256, work.shape, generator=g, device="cuda").to(torch.uint8))
        elif fill != "last":
            work.fill_(fill)
        work[need:] = tail
        out = torch.empty_like(y)
        _native.call("launch_lora_add_kernel", y.data_ptr(), x.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(), scales.data_ptr(), out.data_ptr(),
                     work.data_ptr(), rows, k, n, rank, 5, n, k, n, 1, 2, True, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out, want) and bool((work[need:] == tail).all())


# ------------------------------------------------------------------ large tensors, several callers


def _same(u, v):
    return torch.equal(u.contiguous().view(torch.uint8), v.contiguous().view(torch.uint8))


def test_norm_past_32_bit_offsets(ck):
    g, rows, width = _gen(20), 140001, 16384                               # 2.3 G elements
    x, res, w = (torch.empty(s, dtype=BF16, device="cuda").normal_(generator=g) for s in ((rows, width), (rows, width), (width,)))
    scale = torch.tensor([0.02], device="cuda")
    whole = ck.add_rmsnorm_quantize_mxfp8(x, res, w, return_norm=True)
    fp8 = ck.add_rmsnorm_quantize_fp8(x, res, w, scale)[0]
    for first in (0, 131008, rows - 97):
        part = slice(first, first + 97)
        q, _, h, y = ck.add_rmsnorm_quantize_mxfp8(x[part].clone(), res[part].clone(), w, return_norm=True)
        for got, want in zip((q, h, y), (whole[0], whole[2], whole[3])):
            assert _same(got, want[part])
        assert _same(ck.add_rmsnorm_quantize_fp8(x[part].clone(), res[part].clone(), w, scale)[0], fp8[part])
    assert _same(whole[1], ck.quantize_mxfp8(whole[3])[1])


@pytest.mark.parametrize("tokens_dim", [1, 2])
@pytest.mark.parametrize("unaligned", [0, 1])
def test_rope_past_32_bit_offsets(ck, tokens_dim, unaligned):
    g, n, heads, dim, axes = _gen(21), 140001, 128, 128, (32, 48, 48)
    x = torch.empty(n * heads * dim + unaligned, dtype=BF16, device="cuda").normal_(generator=g)[unaligned:]
    x = x.view((1, n, heads, dim) if tokens_dim == 1 else (1, heads, n, dim))
    pos, freqs = torch.randint(0, 1 << 20, (n, 3), generator=g, device="cuda"), ck.rope_axes_freqs(axes)
    out = ck.apply_rope_axes1(x, pos, freqs, axes, tokens_dim=tokens_dim)
    for first in (0, 131060, n - 40):
        part = slice(first, first + 40)
        cut = lambda t: (t[:, part] if tokens_dim == 1 else t[:, :, part]).contiguous()  # noqa: E731
        if unaligned:     # (the one-pair kernel: the same angles, another order of roundings)
            small = ck.apply_rope_axes1(cut(x), pos[part], freqs, axes, tokens_dim=tokens_dim).double()
            size = cut(x).double().abs().view(*small.shape[:-1], -1, 2).sum(-1, keepdim=True).expand(*small.shape[:-1], -1, 2).reshape(small.shape)
            assert bool(((cut(out).double() - small).abs() <= 2 * (2.0 ** -8 * 1.01 * small.abs() + 2.0 ** -20 * size)).all())
        else:
            assert torch.equal(cut(out), ck.apply_rope_axes1(cut(x), pos[part], freqs, axes, tokens_dim=tokens_dim))


def test_lora_past_32_bit_offsets(ck):
    g, rows, k, n, rank = _gen(22), 300001, 8192, 8200, 24
    x, y = (torch.empty(rows, c, dtype=BF16, device="cuda").normal_(generator=g) for c in (k, n))
    a, b = _randn(g, 5, rank, k, scale=k ** -0.5), _randn(g, 5, n, rank, scale=0.1)
    ids = torch.arange(rows, device="cuda") // 777 % 6
    out = ck.lora_add(y, x, a, b, ids)
    for first in (0, 131000, 262000, rows - 300):
        part = slice(first, first + 300)
        low = torch.stack([x[t].double() @ a[i].double().T if i < 5 else torch.zeros(rank, device="cuda", dtype=torch.float64) for t, i in zip(range(first, first + 300), ids[part].tolist())])
        more = torch.einsum("tr,tnr->tn", low, b.double()[ids[part].clamp(max=4)])
        want = y[part].double() + more
        size = torch.einsum("tr,tnr->tn", low.abs(), b.double().abs()[ids[part].clamp(max=4)])
        # k products of unit variance over sqrt(k) in fp32, then rank; the low-rank vector as two bf16 parts; one rounding to bf16
        bound = 2.0 ** -8 * 1.01 * want.abs() + size * 2.0 ** -16 + (k + rank) * 2.0 ** -23 * k ** 0.5 * b.double().abs().sum(-1).max()
        assert bool(((out[part].double() - want).abs() <= bound).all())
    own = y.clone()
    ck.lora_add(own, x, a, b, ids, out=own)
    assert torch.equal(own, out)


def test_several_threads_at_once(ck):
    """Four threads, each on a stream of its own, with operators of every kind between one another."""
    import threading

    def case(seed):
        g = _gen(seed)
        rows, k, n = 700 + 300 * seed, 512, 1032
        return dict(x=_randn(g, rows, k), y=_randn(g, rows, n), a=_randn(g, 4, 64, k, scale=0.05), b=_randn(g, 4, n, 64, scale=0.1),
                    ids=torch.arange(rows, device="cuda") // (90 + seed) % 5, q=_randn(g, 1, rows, 4, 64), pos=torch.randint(0, 5000, (rows, 2), generator=g, device="cuda"))

    def run(c):
        q, s, h, norm = ck.add_rmsnorm_quantize_mxfp8(c["x"], c["x"], None, return_norm=True)
        few = ck.lora_add(c["y"][:40], norm[:40], c["a"], c["b"], c["ids"][:40])
        return [q, s, h, norm, few, ck.lora_add(c["y"], norm, c["a"], c["b"], c["ids"]), ck.apply_rope_axes1(c["q"], c["pos"], freqs, (24, 40), tokens_dim=1)]

    freqs = ck.rope_axes_freqs((24, 40))
    cases = [case(s) for s in range(4)]
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def worker(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(100):
                    if not all(_same(u, v) for u, v in zip(run(cases[i]), want[i])):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001 - told below
            wrong.append(repr(e))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
