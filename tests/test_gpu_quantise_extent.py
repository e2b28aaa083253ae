"""The quantisers write the bytes of a row and zeros up to the next multiple of 16, whatever the pitch: a destination may be a slice of
a wider matrix."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
KEPT = 0xA5


def pad16(n):
    return (n + 15) // 16 * 16


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 200), (200, 3), (129, 144), (150, 130), (64, 17)])
@pytest.mark.parametrize("pitch", [256, 528])
def test_bytes_behind_a_row_are_left(dtype, M, K, pitch):
    from svoo_b200 import ops
    from svoo_b200._lib import LIB, check
    x = torch.randn(M, K, device=DEV).to(dtype)
    st = torch.cuda.current_stream().cuda_stream
    kb, mb = (K + 127) // 128, (M + 127) // 128
    scales = [torch.empty(n, device=DEV) for n in (kb * M, mb * K, kb * mb)]

    def guarded(rows):
        return torch.full((rows + 1, pitch), KEPT, dtype=torch.uint8, device=DEV)      # a row more than the call is told of

    q = {n: guarded(M) for n in ("rows", "both", "blocks")}
    qt = {n: guarded(K) for n in ("columns", "both", "blocks")}
    head = (x.data_ptr(), ops.TYPES[dtype], M, K, K)
    check(LIB.svoo_b200_quantize_rows(*head, q["rows"].data_ptr(), pitch, scales[0].data_ptr(), M, st), "rows")
    check(LIB.svoo_b200_quantize_columns(*head, qt["columns"].data_ptr(), pitch, scales[1].data_ptr(), K, None, st), "columns")
    check(LIB.svoo_b200_quantize_both(*head, q["both"].data_ptr(), pitch, scales[0].data_ptr(), M, qt["both"].data_ptr(), pitch,
                                      scales[1].data_ptr(), K, None, st), "both")
    check(LIB.svoo_b200_quantize_blocks(*head, q["blocks"].data_ptr(), pitch, qt["blocks"].data_ptr(), pitch, scales[2].data_ptr(), st), "blocks")
    want = {"rows": ops.quantize_rows(x).q, "both": ops.quantize_rows(x).q, "blocks": ops.quantize_blocks(x).q}
    want_t = {"columns": ops.quantize_columns(x).q, "both": ops.quantize_columns(x).q, "blocks": ops.quantize_blocks(x, True).qt}
    for got, ref in [(q[n], want[n]) for n in q] + [(qt[n], want_t[n]) for n in qt]:
        rows, cols = ref.shape
        assert torch.equal(got[:rows, :cols], ref.view(torch.uint8))
        assert not got[:rows, cols:pad16(cols)].any()
        assert (got[:rows, pad16(cols):] == KEPT).all() and (got[rows] == KEPT).all()


@pytest.mark.parametrize("M,N,K", [(5, 77, 200), (40, 300, 136), (40, 72, 1000), (9600, 270, 128), (9600, 513, 130)])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32", "e4m3", "e4m3 gelu"])
def test_results_in_a_wider_matrix(M, N, K, kind):
    """Products of few tiles and of many, and the call on unquantised rows: nothing is written behind a row of the result (an e4m3 row
    ends at the next multiple of 16), behind its last row, or behind its scales."""
    from svoo_b200 import ops
    from svoo_b200._lib import LIB, check
    number = {"bf16": 0, "fp16": 1, "fp32": 2}.get(kind, 3)
    dtype = [torch.bfloat16, torch.float16, torch.float32, torch.uint8][number]
    e4m3, gelu = number == 3, kind.endswith("gelu")
    x, b = torch.randn(M, K, device=DEV).bfloat16(), ops.quantize_blocks(torch.randn(N, K, device=DEV))
    bias = torch.randn(N, device=DEV)
    a = ops.quantize_rows(x)
    st = torch.cuda.current_stream().cuda_stream
    nb, pitch_s = (N + 127) // 128, M + 3
    ws = torch.empty(M * pad16(K) + 256 + 4 * M * ((K + 127) // 128), dtype=torch.uint8, device=DEV)
    for pitch in ([pad16(N), pad16(N) + 64] if e4m3 else [N, N + 3, pad16(N) + 32]):
        for whole in (False, True):
            out = torch.zeros(M + 1, pitch, dtype=dtype, device=DEV)
            out.view(torch.uint8).fill_(KEPT)
            kept = out[-1].clone()
            scale = torch.full((nb + 1, pitch_s), -7.0, device=DEV)
            tail = (bias.data_ptr(), 2)
            end = (int(gelu), out.data_ptr(), number, pitch, scale.data_ptr() if e4m3 else None, pitch_s)
            if whole:
                check(LIB.svoo_b200_linear_fp8(x.data_ptr(), 0, M, K, K, b.q.data_ptr(), pad16(K), b.scale.data_ptr(), *b.scale.stride(), *tail, N, *end,
                                               ws.data_ptr(), ws.numel(), st), "linear_fp8")
                ref = ops.linear_fp8(x, b, bias, "gelu" if gelu else None, ops.E4M3 if e4m3 else dtype)
            else:
                check(LIB.svoo_b200_mm_fp8(a.q.data_ptr(), pad16(K), a.scale.data_ptr(), M, b.q.data_ptr(), pad16(K), b.scale.data_ptr(), *b.scale.stride(),
                                           0, *tail, M, N, K, *end, st), "mm_fp8")
                ref = ops.mm_fp8(a, b, bias, "gelu" if gelu else None, ops.E4M3 if e4m3 else dtype)
            cols = pad16(N) if e4m3 else N
            if e4m3:
                assert torch.equal(scale[:nb, :M], ref.scale) and (scale[:, M:] == -7).all() and (scale[nb] == -7).all()
                assert not out[:M, N:cols].any()
                ref = ref.q.view(torch.uint8)
            assert torch.equal(out[:M, :N], ref)
            assert (out[:M, cols:].contiguous().view(torch.uint8) == KEPT).all()
            assert torch.equal(out[M].view(torch.uint8), kept.view(torch.uint8))
