"""Host-compiled checks of rules the kernels share with the host: small programs around the headers of csrc/,
built with nvcc and run on the CPU."""
import os
import subprocess

from svoo_b200 import build

MAP_READS = r"""
#include <cstdio>
#include "map_common.cuh"
// Every read, at every alignment of maps of 1 to 5 rows: it lies inside the map, and the bytes are the map's.
struct Recorder {
  const uint8_t *lo, *hi;
  mutable bool outside = false;
  uint32_t word(const uint8_t* p) const {
    outside |= p < lo || p + 4 > hi || reinterpret_cast<uintptr_t>(p) % 4;
    return p[0] | p[1] << 8 | p[2] << 16 | (uint32_t)p[3] << 24;
  }
  uint32_t byte(const uint8_t* p) const {
    outside |= p < lo || p >= hi;
    return *p;
  }
};
int main() {
  alignas(8) static uint8_t mem[4096];
  const int rows_of[] = {1, 2, 5}, cols_of[] = {1, 2, 3, 4, 5, 31, 32, 33, 63, 65, 97, 500};
  for (int rows : rows_of)
    for (int KC : cols_of)
      for (int place = 64; place < 68; ++place) {
        const int total = rows * KC;
        uint8_t* map = mem + place;
        for (int i = 0; i < total; ++i) map[i] = (uint8_t)(i * 37 % 3);
        const Recorder load{map, map + total};
        for (int r = 0; r < rows; ++r)
          for (int lane = 0; lane < 32; ++lane) {
            const int j0 = lane * 32, left = KC - j0, bytes = left < 0 ? 0 : (left > 32 ? 32 : left);
            uint32_t w[9];
            const int skew = svoo::map_words(w, map + r * KC + j0, bytes, map, map + total, load);
            for (int b = 0; b < bytes; ++b)
              if ((w[(b + skew) / 4] >> (8 * ((b + skew) % 4)) & 0xFF) != map[r * KC + j0 + b]) return printf("wrong byte\n"), 1;
          }
        if (load.outside) return printf("read outside: %d x %d at %d\n", rows, KC, place), 1;
      }
  puts("ok");
  return 0;
}
"""


SORT_RULE = r"""
#include <cstdio>
#include "common.cuh"
// The sort takes the largest cluster that the size asks for and the device can place.
int main() {
  const long sizes[][3] = {{1, 1, 1}, {2, 4096, 32}, {12, 32760, 500}, {40, 75600, 500}, {3, 40003, 1024}, {64, 75600, 100}, {300, 75600, 100}};
  const int want[] = {1, 8, 16, 8, 16, 8, 1};
  for (int i = 0; i < 7; ++i)
    for (int limit = 1; limit <= 16; limit *= 2) {
      const int got = svoo::sort_cluster_ctas(sizes[i][0], sizes[i][1], sizes[i][2], 148, [&](int ctas) { return ctas <= limit; });
      if (got != (want[i] < limit ? want[i] : limit)) return printf("%d %d: %d\n", i, limit, got), 1;
    }
  puts("ok");
  return 0;
}
"""


def _run(tmp_path, source):
    src, exe = tmp_path / "t.cu", tmp_path / "t"
    src.write_text(source)
    res = subprocess.run([build._nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", build.CSRC,
                          str(src), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", (out.returncode, out.stdout)


def test_map_words_stay_inside_the_map(tmp_path):
    _run(tmp_path, MAP_READS)


def test_sort_takes_a_cluster_that_fits(tmp_path):
    _run(tmp_path, SORT_RULE)


def test_token_wise_entry_points_check_their_arguments():
    """Layer norm, quantisers and 8-bit products refuse bad arguments on the host; nothing is launched."""
    import ctypes
    from svoo_b200._lib import LIB as L
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    norm = lambda **k: L.svoo_b200_layer_norm(*[{**dict(x=p, t=0, b=1, r=2, C=64, xb=128, xr=64, g=p, gb=0, o=p, ob=0, pt=2, one=0, eps=1e-6,  # noqa: E731
                                                         y=p, m=None, s=None, st=None), **k}[n] for n in
                                                 ("x", "t", "b", "r", "C", "xb", "xr", "g", "gb", "o", "ob", "pt", "one", "eps", "y", "m", "s", "st")])
    assert norm(r=0) == 0 and norm(b=0) == 0
    assert norm(x=None) == -1 and norm(y=None) == -1 and norm(m=p) == -1
    assert norm(C=0) == -2 and norm(C=16385) == -2 and norm(r=-1) == -2 and norm(xr=-1) == -2 and norm(b=1 << 20, r=1 << 20) == -2
    assert norm(b=70000, r=1, gb=64) == -2 and norm(b=1 << 11, r=1 << 20) == -2
    assert norm(t=3) == -8 and norm(t=0, pt=1) == -8
    assert norm(x=p + 1) == -5 and norm(g=p + 2) == -5
    out = ctypes.c_int64(0)
    assert L.svoo_b200_layer_norm_workspace_bytes(2, 100, 64, 1, ctypes.byref(out)) == 0 and out.value >= 2 * 2 * 64 * 4
    assert L.svoo_b200_layer_norm_workspace_bytes(70000, 100, 64, 1, ctypes.byref(out)) == -2
    assert L.svoo_b200_layer_norm_workspace_bytes(2, 100, 64, 1, None) == -1
    back = lambda ws, dg, do: L.svoo_b200_layer_norm_backward(p, 0, 64, p, 0, 1, 2, 64, 0, 64, p, p, p, 0, 2, 0, 0, p, dg, do, p, ws, None)  # noqa: E731
    assert back(1 << 20, p, None) == -1 and back(4, p, p) == -4
    assert L.svoo_b200_quantize_rows(p, 0, 4, 100, 100, p, 100, p, 4, None) == -2        # pitch not a multiple of 16
    assert L.svoo_b200_quantize_rows(p, 0, 4, 100, 100, p, 96, p, 4, None) == -2
    assert L.svoo_b200_quantize_rows(p, 0, 4, 100, 100, p, 112, p, 3, None) == -2
    assert L.svoo_b200_quantize_rows(p, 3, 4, 100, 100, p, 112, p, 4, None) == -8
    assert L.svoo_b200_quantize_rows(p, 0, 4, 100, 100, p + 8, 112, p, 4, None) == -5
    assert L.svoo_b200_quantize_rows(p, 0, 0, 100, 100, None, 112, None, 0, None) == 0
    assert L.svoo_b200_quantize_columns(p, 0, 100, 4, 4, p, 96, p, 4, None, None) == -2
    assert L.svoo_b200_quantize_blocks(p, 0, 100, 4, 4, p, 16, p, 96, p, None) == -2
    assert L.svoo_b200_quantize_blocks(p, 0, 100, 4, 4, p, 16, p + 1, 112, p, None) == -5
    assert L.svoo_b200_column_sum(p, -1, 4, p, 2, None) == -2 and L.svoo_b200_column_sum(p, 1, 4, None, 2, None) == -1
    d = dict(a=p, ap=64, sa=p, sap=8, b=p, bp=64, sb=p, sn=1, sk=1, rows=0, bias=None, bt=0, M=8, N=16, K=64, act=0, out=p, ot=0, op=16, os=None,
             osp=0, st=None)
    mm = lambda **k: L.svoo_b200_mm_fp8(*{**d, **k}.values())                             # noqa: E731
    assert mm(M=0) == 0
    assert mm(a=None) == -1 and mm(out=None) == -1 and mm(ot=3) == -2 and mm(ot=3, op=16, osp=8) == -1
    assert mm(K=0) == -2 and mm(N=0) == -2 and mm(ap=72) == -2 and mm(ap=48) == -2 and mm(sap=7) == -2 and mm(op=15) == -2
    assert mm(rows=1, sk=12) == -2 and mm(rows=1, sk=18) == -2 and mm(rows=1, sk=16, act=1) == -8 and mm(rows=1, sk=16, ot=3) == -8
    assert mm(act=2) == -8 and mm(ot=4) == -8 and mm(bias=p, bt=3) == -8
    assert mm(a=p + 8) == -5 and mm(rows=1, sk=16, sb=p + 4) == -5
    assert L.svoo_b200_linear_status(None, None) == -1
    assert L.svoo_b200_linear_fp8_workspace_bytes(16, 100, 0, ctypes.byref(out)) == 0 and out.value == 0
    assert L.svoo_b200_linear_fp8_workspace_bytes(16, 100, 3, ctypes.byref(out)) == 0 and out.value >= 16 * 112 + 64
    assert L.svoo_b200_linear_fp8_workspace_bytes(17, 100, 0, ctypes.byref(out)) == 0 and out.value >= 17 * 112 + 68
    assert L.svoo_b200_linear_fp8_workspace_bytes(9, 5000, 0, ctypes.byref(out)) == 0 and out.value >= 9 * 5008
    few = dict(x=p, t=0, M=4, K=64, xr=64, b=p, bp=64, sb=p, sn=1, sk=1, bias=None, bt=0, N=16, act=0, out=p, ot=0, op=16, os=None, osp=4, ws=None,
               wb=0, st=None)
    lin = lambda **k: L.svoo_b200_linear_fp8(*{**few, **k}.values())                      # noqa: E731
    assert lin(M=0) == 0 and lin(x=None) == -1 and lin(b=None) == -1 and lin(out=None) == -1 and lin(bp=72) == -2 and lin(t=3) == -8
    assert lin(M=17) == -1 and lin(M=17, ws=p, wb=16) == -4 and lin(ot=3) == -1 and lin(K=0) == -2 and lin(b=p + 8) == -5
    three = (ctypes.c_int64 * 3)()
    assert L.svoo_b200_linear_train_bytes(100, 200, 300, 1, 1, three) == 0 and all(v > 0 for v in three)
    whole = list(three)
    assert L.svoo_b200_linear_train_bytes(100, 200, 300, 0, 0, three) == 0 and three[0] < whole[0] and list(three)[1:] == whole[1:]
    assert L.svoo_b200_linear_train_bytes(0, 200, 300, 1, 1, three) == -2 and L.svoo_b200_linear_train_bytes(1, 1, 1, 1, 1, None) == -1
    fw = dict(x=p, t=0, M=4, K=64, xr=64, w=p, wt=0, N=16, wr=64, bias=None, bt=0, kx=1, kw=1, y=p, sv=p, sb=1 << 20, ws=p, wb=1 << 20, st=None)
    forward = lambda **k: L.svoo_b200_linear_train_forward(*{**fw, **k}.values())         # noqa: E731
    assert forward(x=None) == -1 and forward(sv=None) == -1 and forward(t=3) == -8 and forward(wt=4) == -8 and forward(M=0) == -2
    assert forward(sb=64) == -4 and forward(wb=64) == -4 and forward(sv=p + 8) == -5 and forward(bias=p, bt=3) == -8 and forward(xr=-1) == -2
    bwd = dict(dy=p, t=0, M=4, N=16, K=64, r=16, sv=p, sb=1 << 20, kx=1, kw=1, dx=p, dw=p, wt=0, db=p, bt=0, ws=p, wb=1 << 20, st=None)
    backward = lambda **k: L.svoo_b200_linear_train_backward(*{**bwd, **k}.values())      # noqa: E731
    assert backward(dx=None, dw=None, db=None) == 0
    assert backward(dy=None) == -1 and backward(kx=0) == -1 and backward(kw=0) == -1 and backward(wt=3) == -8 and backward(bt=3) == -8
    assert backward(sb=64) == -4 and backward(wb=64) == -4 and backward(dy=p + 1) == -5 and backward(N=0) == -2


def test_product_kernels_do_not_spill():
    """tcgen05.ld fills registers behind the instruction stream: code that issues it must not spill (a register could be saved
    before it is filled).  The register shares that setmaxnreg deals out add up to a launch at 168 registers a thread."""
    import os
    import re
    import subprocess
    from svoo_b200 import build
    for src, kernels in (("linear_tc.cu", 11), ("linear_split.cu", 8)):
        res = subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xptxas", "-v", "-c",
                              os.path.join(build.CSRC, src), "-o", os.devnull], capture_output=True, text=True)
        assert res.returncode == 0, res.stderr
        spills = re.findall(r"(\d+) bytes spill stores, (\d+) bytes spill loads", res.stderr)
        assert len(spills) >= kernels and all(s == ("0", "0") for s in spills), res.stderr
        if src == "linear_tc.cu":
            assert set(re.findall(r"Used (\d+) registers", res.stderr)) == {"168"}


def test_token_kernels_need_a_model_on_its_gpu():
    """Refused before anything of the model is changed."""
    import pytest
    import torch
    from svoo_b200 import wan_dit
    cfg = wan_dit.WanDiTConfig(num_layers=1, dim=128, heads=1, ffn_dim=128, text_dim=16, text_len=4, latent=(1, 4, 4))
    model = wan_dit.WanDiT(cfg)
    with pytest.raises(ValueError, match="GPU"):
        model.use_token_kernels()
    assert not model.blocks[0].fused_norms and isinstance(model.blocks[0].attn1.to_q, torch.nn.Linear)


def test_gradient_of_samples_with_gains_of_their_own():
    """Shared sums of gains that differ by sample are refused on the host, as are more such samples than the grid has."""
    import ctypes
    from svoo_b200._lib import LIB as L
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    back = lambda b, gb, per, dg: L.svoo_b200_layer_norm_backward(p, 128, 64, p, 0, b, 2, 64, 128, 64, p, p, p, gb, 2, 1, per, p, dg, dg, p, 4, None)  # noqa: E731
    assert back(2, 64, 0, p) == -2 and back(2, 64, 1, p) == -4 and back(2, 0, 0, p) == -4 and back(1, 64, 0, p) == -4
    assert back(70000, 64, 0, None) == -2 and back(70000, 64, 1, p) == -2


def test_a_model_reports_token_kernels_that_gave_up(monkeypatch):
    """check_status asks every processor, and the token-wise kernels of the model's device once blocks are on them; it raises."""
    import pytest
    import torch
    from svoo_b200 import linear, ops, wan_dit
    cfg = wan_dit.WanDiTConfig(num_layers=2, dim=128, heads=1, ffn_dim=128, text_dim=16, text_len=4, latent=(1, 4, 4))
    model = wan_dit.WanDiT(cfg)
    asked, word = [], [0]

    class Processor:
        def check_status(self):
            asked.append("processor")

    def status(device):
        asked.append(device)
        return word[0]

    monkeypatch.setattr(ops, "linear_status", status)
    model.blocks[1].attn1.set_processor(Processor())
    model.check_status()
    assert asked == ["processor"]
    model.blocks[1].fused_norms = True
    model.check_status()
    assert asked == ["processor"] * 2 + [torch.device("cpu")]
    word[0] = 1
    with pytest.raises(RuntimeError, match="incomplete"):
        model.check_status()
    model.blocks[1].fused_norms = False
    model.check_status()
    model.blocks[0].attn2.to_k = linear.Fp8Linear(128, 128)   # one layer, put there by hand
    with pytest.raises(RuntimeError, match="incomplete"):
        model.check_status()


def test_forward_mode_is_refused():
    """A tangent on any tensor of a call raises before anything else is looked at; without one the call gets to its other checks."""
    import pytest
    import torch
    from torch.autograd import forward_ad
    from svoo_b200 import linear, norm
    x, w, v = torch.randn(4, 8), torch.randn(8, 8), torch.randn(8)
    stored = linear.Fp8Weight(w.to(torch.float8_e4m3fn), torch.ones(1, 1))
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, v)]
        for fn, args in ((norm.layer_norm, (dual[0],)), (norm.layer_norm, (x, dual[2], v)), (norm.layer_norm, (x, v, dual[2])),
                         (linear.linear_fp8, (dual[0], w)), (linear.linear_fp8, (x, dual[1])), (linear.linear_fp8, (x, w, dual[2])),
                         (linear.linear_fp8, (dual[0], stored)), (linear.mlp_fp8, (dual[0], stored, v, stored, v)),
                         (linear.mlp_fp8, (x, stored, v, stored, dual[2]))):
            with pytest.raises(NotImplementedError):
                fn(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                fn(*args)
        with pytest.raises(ValueError, match="CUDA"):
            norm.layer_norm(x, v, v)
    with pytest.raises(ValueError, match="CUDA"):
        linear.linear_fp8(x, w)


def test_norm_kernels_are_those_that_sizes_choose():
    """The library holds a norm kernel for a type, alignment and number of pieces and threads only where some number of columns takes it."""
    import re
    names = subprocess.run(["nm", "-C", build.build()], capture_output=True, text=True).stdout
    held = {(d or "", t, int(nv), int(tpr), al == "true") for d, t, nv, tpr, al in
            re.findall(r"layer_norm(_backward)?_ring_kernel<(\w+), (\d+), (\d+), (true|false)>", names)}
    chosen = set()
    for t, e in (("__nv_bfloat16", 2), ("__half", 2), ("float", 4)):
        per_piece = 16 // e
        for aligned in (True, False):
            for C in range(1, 16385):
                if aligned and C * e % 16:
                    continue
                pieces, unit = -(-C // per_piece), 8 // per_piece
                tpr = 32 if C <= 2048 else 64 if C <= 5120 else 128 if C <= 8192 else 256
                steps = {32: (2, 4, 6, 8), 64: (6, 10), 128: (8,), 256: (8,)}[tpr]
                chosen.add(("", t, min(n * unit for n in steps if n * unit * tpr >= pieces), tpr, aligned))
                wide = C * (e if aligned else 4)
                tpr = 32 if wide <= 2560 else 64 if wide <= 5120 else 128 if wide <= 10240 else 256
                chosen.add(("_backward", t, min(n * unit for n in (3, 5, 8) if n * unit * tpr >= pieces), tpr, aligned))
    assert held == chosen, held ^ chosen
