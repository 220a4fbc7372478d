"""A 4-bit product one of whose copies never arrives: the bounded wait runs out (2 s), the outputs whose sums lack a part
come out as NaN, all others as ever, and the status words say so.  The kernel is compiled here with a copy that
leaves one unit out; the library's own call and its check are asked beside it."""
import subprocess

import pytest

from conftest import PKG_DIR, ROOT

pytestmark = pytest.mark.gpu

PROGRAM = r"""
#include <cuda_runtime.h>
#include <cstdio>
#include <cstring>
#include <vector>
#include "gemv_w4.cuh"
using namespace qasr;

__device__ int lose_tile, lose_unit;
struct Losing {
  static __device__ void unit(void* slot, const uint8_t* from, uint32_t bytes, uint64_t* full, int tile, int unit) {
    if (tile == lose_tile && unit == lose_unit) return;
    W4Copy::unit(slot, from, bytes, full, tile, unit);
  }
};

// tiles x units, CTAs, CTAs per cluster, the unit that is lost (tile -1: none)
static std::vector<uint16_t> run(int tiles, int units, int ctas, int cluster, int tile, int unit, int accumulate, uint32_t* status) {
  const int n_out = tiles * 32, k = units * 128, rows = 3;
  std::vector<uint8_t> codes(size_t(n_out) * k / 2);
  for (size_t i = 0; i < codes.size(); ++i) codes[i] = uint8_t(i * 2654435761u >> 13);
  std::vector<uint16_t> scale(size_t(n_out) * units, 0x2000), x(size_t(rows) * k), out(size_t(rows) * n_out, 0x3c00);  // 2^-7; 1
  for (size_t i = 0; i < x.size(); ++i) x[i] = uint16_t(0x3800 + i % 1024) | uint16_t(i % 3 ? 0x8000 : 0);
  const W4Layout L = w4_layout(n_out, k, 128, false);
  uint8_t *d_codes, *d_packed;
  uint16_t *d_scale, *d_x, *d_out;
  cudaMalloc(&d_codes, codes.size());
  cudaMalloc(&d_scale, scale.size() * 2);
  cudaMalloc(&d_packed, L.total);
  cudaMalloc(&d_x, x.size() * 2);
  cudaMalloc(&d_out, out.size() * 2);
  cudaMemcpy(d_codes, codes.data(), codes.size(), cudaMemcpyHostToDevice);
  cudaMemcpy(d_scale, scale.data(), scale.size() * 2, cudaMemcpyHostToDevice);
  cudaMemcpy(d_x, x.data(), x.size() * 2, cudaMemcpyHostToDevice);
  cudaMemcpy(d_out, out.data(), out.size() * 2, cudaMemcpyHostToDevice);
  pack_w4_kernel<<<8, 256>>>(d_codes, d_scale, nullptr, n_out, k, 128, d_packed);
  cudaMemcpyToSymbol(lose_tile, &tile, 4);
  cudaMemcpyToSymbol(lose_unit, &unit, 4);
  const uint32_t none[2] = {0, 0};
  cudaMemcpyToSymbol(w4_status, none, 8);
  const auto kernel = gemv_w4_kernel<false, false, 1, 1, Losing>;
  using P = W4Plan<false, 1, 1>;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::smem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(W4_THREADS);
  cfg.dynamicSmemBytes = P::smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1;
  const W4Args a{d_packed, n_out, k, d_x, k, rows, d_out, n_out, accumulate, 3, cluster};
  cudaLaunchKernelEx(&cfg, kernel, a);
  cudaMemcpyFromSymbol(status, w4_status, 8);
  cudaMemcpy(out.data(), d_out, out.size() * 2, cudaMemcpyDeviceToHost);
  if (cudaError_t e = cudaDeviceSynchronize()) std::printf("cuda: %s\n", cudaGetErrorString(e));
  cudaFree(d_codes); cudaFree(d_scale); cudaFree(d_packed); cudaFree(d_x); cudaFree(d_out);
  return out;
}

int main() {
  struct Case { int tiles, units, ctas, cluster, tile, unit, accumulate, first, last; };  // tiles [first, last) must be NaN
  const Case cases[] = {
      {3, 8, 3, 1, 1, 5, 0, 1, 2},    // a CTA per tile
      {3, 8, 3, 1, 2, 0, 1, 2, 3},    // added to what is there
      {4, 16, 1, 1, 1, 12, 1, 1, 4},  // one CTA for all: the warp that gave up has no part in the later tiles either
      {2, 64, 4, 2, 1, 40, 0, 1, 2},  // two CTAs of a cluster share a tile; the second one's part is lost
  };
  int bad = 0, n = 0;
  for (const Case& c : cases) {
    uint32_t clean_status[2], status[2];
    const auto clean = run(c.tiles, c.units, c.ctas, c.cluster, -1, 0, c.accumulate, clean_status);
    const auto lost = run(c.tiles, c.units, c.ctas, c.cluster, c.tile, c.unit, c.accumulate, status);
    int wrong = 0;
    for (size_t i = 0; i < clean.size(); ++i) {
      const int tile = int(i % (c.tiles * 32)) / 32;
      const bool nan = (lost[i] & 0x7fff) > 0x7c00, want = tile >= c.first && tile < c.last;
      wrong += want ? !nan : lost[i] != clean[i];
      wrong += (clean[i] & 0x7fff) >= 0x7c00;
    }
    if (wrong || clean_status[0] || status[0] != DEVERR_TIMEOUT || status[1] != W4_WAIT_SITE) bad |= 1 << n;
    std::printf("case %d: %d wrong, status %u %u (clean %u)\n", n++, wrong, status[0], status[1], clean_status[0]);
  }
  return bad;
}
"""


def test_a_copy_that_never_arrives(cuda_device, tmp_path):
    src, exe = tmp_path / "lost.cu", tmp_path / "lost"
    src.write_text(PROGRAM)
    subprocess.run(["/usr/local/cuda/bin/nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                    "--expt-relaxed-constexpr", "-I", str(PKG_DIR / "csrc"), "-I", str(ROOT / "include"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


def test_w4_check_finds_nothing_after_good_calls(qasr, cuda_device):
    import torch

    from test_gpu_serving_ops import W4, _stream
    w = W4(qasr, torch, 300, 2048, 64, True, "f16", 5)
    for _ in range(3):
        w.run(qasr)
    qasr.kernel_gemv_w4_check(0, _stream(torch))
    w.check(w.out)
    with pytest.raises(qasr.DecoderError):
        qasr.kernel_gemv_w4_check(99, 0)
