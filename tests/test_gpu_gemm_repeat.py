"""The block-scaled GEMM gives the same result every time.

Its two MMA issuers take the k-tiles in turn; with one full barrier for a stage an issuer could take an older phase for its own when
copies landed late, and about one launch in 2000 had a wrong tile.  So: many launches in a row, one result.  (Not always the same
bits: which issuer's MMA enters the pipe first is not fixed, and the order of a sum shows in its last bit.)
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

LAUNCHES = 2000


def _operands(kind, m, n, k):
    """(a GEMM, the largest sum of its products' absolute values)"""
    import comfy_kitchen as ck

    g = torch.Generator(device="cuda").manual_seed(k)
    x, w = (torch.randn(r, k, generator=g, device="cuda").bfloat16() for r in (m, n))
    if kind == "mxfp8":
        (qx, sx), (qw, sw) = ck.quantize_mxfp8(x), ck.quantize_mxfp8(w)
        size = ck.dequantize_mxfp8(qx, sx, torch.float32).abs() @ ck.dequantize_mxfp8(qw, sw, torch.float32).abs().T
        return (lambda: ck.scaled_mm_mxfp8(qx, qw, sx, sw, out_dtype=torch.bfloat16)), size.max().item()
    ts = torch.full((1,), 0.002, device="cuda")
    (qx, sx), (qw, sw) = ck.quantize_nvfp4(x, ts), ck.quantize_nvfp4(w, ts)
    size = ck.dequantize_nvfp4(qx, ts, sx, torch.float32).abs() @ ck.dequantize_nvfp4(qw, ts, sw, torch.float32).abs().T
    return (lambda: ck.scaled_mm_nvfp4(qx, qw, ts, ts, sx, sw, out_dtype=torch.bfloat16)), size.max().item()


# 18 x 36 tiles for 74 pairs of CTAs.  K: an even number of k-tiles, and an odd one (the issuer that opens a tile alternates), of
# 128 (MXFP8) or of 256 (NVFP4) elements, the last one whole and not
@pytest.mark.parametrize("kind,k", [("mxfp8", 4096), ("mxfp8", 2944), ("mxfp8", 2848), ("nvfp4", 4096), ("nvfp4", 2816), ("nvfp4", 2784)])
def test_same_result_every_time(kind, k):
    call, size = _operands(kind, 4608, 9216, k)
    first = call()
    # k roundings of a sum in fp32, in either launch; then a rounding to bf16 of each, and one of their difference
    bound = (2 * k * 2.0 ** -24 * size + 2 * 2.0 ** -8 * first.abs().max().item()) * (1 + 2.0 ** -8)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(LAUNCHES):
        wrong += ~((call() - first).abs().amax() <= bound)
    # (a wrong k-tile is 128 products or more of unit variance taken for others: a difference of 16 on average over 65536 elements)
    assert bound < 16 and wrong.item() == 0
    from comfy_kitchen.backends import cuda

    assert cuda.gemm_device_status() == 0
