"""Results of the GEMM kernels in fp32."""
import pytest
import torch

from test_gemm_gpu import _rand

pytestmark = pytest.mark.gpu


def _check(got, a, w):
    """A product of bf16 numbers is exact in fp32; an accumulator takes sixteen of them at a time, of which each, and the sum before, may be cut
    at 2^-23 of the largest: at most 17 / 16 K 2^-23 of the sum of magnitudes, bounded by K 2^-22."""
    assert got.dtype == torch.float32
    want, mag = a.double() @ w.double().T, a.double().abs() @ w.double().abs().T
    assert ((got.double() - want).abs() <= a.shape[1] * 2.0 ** -22 * mag).all()


@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (128, 256, 64), (9, 4096, 1024), (200, 264, 328), (384, 776, 512), (513, 9000, 256), (2048, 4096, 256)])
@pytest.mark.parametrize("tile_n,pair", [(0, 0), (128, -1), (256, -1), (128, 0), (256, 0)])
def test_gemm_f32(M, N, K, tile_n, pair):
    from mesh_b200.ops.gemm import gemm
    from mesh_b200.utils.status import check_status
    a, w = _rand((M, K), seed=1), _rand((N, K), seed=2)
    got = gemm(a, w, out_f32=True, tile_n=tile_n, pair=pair)
    check_status()
    _check(got, a, w)
    assert torch.equal(got.to(torch.bfloat16), gemm(a, w, tile_n=tile_n, pair=pair))          # the accumulators are the same


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N,K", [(9, 4096, 512), (200, 264, 320), (513, 2056, 256)])
def test_gemm_q_f32(bits, M, N, K):
    from mesh_b200.ops import decode as D
    from mesh_b200.ops.gemm import gemm_q
    from mesh_b200.utils.status import check_status
    quantize, dequantize = (D.quantize_w4, D.dequantize_w4) if bits == 4 else (D.quantize_w8, D.dequantize_w8)
    a = _rand((M, K), seed=3)
    codes, scales = quantize(_rand((N, K), 0.05, seed=4))
    # the weights that go into the products: of 4-bit codes bf16(bf16(scale) * code), of 8-bit ones bf16(scale * code)
    w = dequantize(codes, scales.bfloat16() if bits == 4 else scales)
    for tile_n, pair in ((0, 0), (128, -1), (256, -1), (128, 0), (256, 0)):
        got = gemm_q(a, codes, scales, out_f32=True, tile_n=tile_n, pair=pair)
        check_status()
        _check(got, a, w)
        assert torch.equal(got.to(torch.bfloat16), gemm_q(a, codes, scales, tile_n=tile_n, pair=pair))


def test_gemm_f32_into_part_of_a_matrix():
    from mesh_b200.ops.gemm import gemm
    a, w = _rand((70, 64), seed=5), _rand((40, 64), seed=6)
    room = torch.full((72, 60), 5.0, device="cuda")
    out = room[1:71, 4:44]
    assert gemm(a, w, out=out, out_f32=True) is out
    _check(out, a, w)
    room[1:71, 4:44] = 5
    assert (room == 5).all()


def test_gemm_f32_refusals():
    from mesh_b200.ops.gemm import gemm
    a, w = _rand((64, 64), seed=5), _rand((64, 64), seed=6)
    for kw in (dict(a_mn=True), dict(b_mn=True), dict(out=torch.empty(64, 64, device="cuda", dtype=torch.bfloat16)), dict(out=torch.empty(64, 72, device="cuda")),
               dict(out=torch.empty(63, 64, device="cuda")), dict(out=torch.empty(64, 64)), dict(out=torch.empty(64, 64, device="cuda").t()[:, ::1])):
        with pytest.raises(ValueError):
            gemm(a, w, out_f32=True, **kw)
    for out in (torch.empty(64, 66, device="cuda")[:, :64], torch.empty(64, 68, device="cuda")[:, 1:65]):
        with pytest.raises(RuntimeError, match="fp32 D"):
            gemm(a, w, out_f32=True, out=out)
