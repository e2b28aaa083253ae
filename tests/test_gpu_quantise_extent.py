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
