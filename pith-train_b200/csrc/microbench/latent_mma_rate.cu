// Micro-benchmark behind the latent attention kernel's design notes: how many cycles a tcgen05.mma of few columns takes when
// one lane issues them back to back, with A (128 rows) from shared memory as the kernel's tiles lie there.
//
//   nvcc -gencode arch=compute_100a,code=sm_100a -O3 -std=c++17 -I.. -I../../../include \
//        -o latent_mma_rate latent_mma_rate.cu ../host_common.cu && ./latent_mma_rate
//
// kind::f16 (bf16, K = 16) and kind::f8f6f4 (e4m3, K = 32), A K-major (score GEMM) or MN-major (output GEMM). Every wait is
// bounded. Not part of the library: nothing links or imports it.
#include <cstdio>
#include "common.cuh"
#include "host_common.h"
using namespace pith;

constexpr int kSmem = 176 * 1024, kB = 128 * 1024;  // A: four blocks of 128 x 128 bytes behind offset 0; B: N x 256 bytes

__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int N, bool MN, bool FP8>
__global__ void __launch_bounds__(128, 1) rate_kernel(long long* out, int reps) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bar;
  __shared__ uint32_t slot, aflag;
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kSmem / 4; i += 128) reinterpret_cast<uint32_t*>(smem)[i] = 0;
  if (threadIdx.x == 0) {
    aflag = 0;
    mbar_init(&bar, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&slot, 512);
    tmem_relinquish();
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = slot;
  const AbortCtl ctl{nullptr, &aflag};
  if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t idesc = FP8 ? (1u << 4) | (static_cast<uint32_t>(MN) << 15) | (static_cast<uint32_t>(N >> 3) << 17) | (8u << 24)
                                   : make_idesc_bf16(128, N, MN, false);
    const uint64_t ad = make_smem_desc(smem_u32(smem), MN ? 16384 : 16, 1024);
    const uint64_t bd = make_smem_desc(smem_u32(smem) + kB, 16, 1024);
    const long long t0 = clock64();
    for (int r = 0; r < reps; ++r) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t at = !MN ? (k >> 2) * 16384 + (k & 3) * 32 : FP8 ? (k >> 2) * 16384 + (k & 3) * 4096 : k * 2048;
        const uint64_t a = desc_advance(ad, at), b = desc_advance(bd, (k >> 2) * (N * 128) + (k & 3) * 32);
        if (leader) {
          if (FP8) mma_e4m3(tmem, a, b, idesc, k > 0);
          else umma_ss(tmem, a, b, idesc, k > 0);
        }
      }
    }
    if (leader) umma_commit(&bar);
    mbar_wait(&bar, 0, ctl, 1);
    if (blockIdx.x == 0 && leader) *out = clock64() - t0;
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <int N, bool MN, bool FP8>
static int rate() {
  static_assert(kB + N * 256 <= kSmem, "shared memory");
  long long *d = nullptr, h = 0;
  auto kernel = rate_kernel<N, MN, FP8>;
  const int reps = 64;
  cudaMalloc(&d, sizeof h);
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  for (int i = 0; i < 3; ++i) kernel<<<148, 128, kSmem>>>(d, reps);
  const cudaError_t e = cudaDeviceSynchronize();
  cudaMemcpy(&h, d, sizeof h, cudaMemcpyDeviceToHost);
  cudaFree(d);
  printf("%s, A %s-major, N %3d: %6.1f cycles per MMA  %s\n", FP8 ? "e4m3 K 32" : "bf16 K 16", MN ? "MN" : "K ", N,
         double(h) / (8 * reps), cudaGetErrorString(e));
  return e != cudaSuccess;
}

int main() {
  return rate<16, false, false>() | rate<32, false, false>() | rate<64, false, false>() | rate<128, false, false>() |
         rate<16, true, false>() | rate<32, true, false>() | rate<64, true, false>() | rate<128, true, false>() |
         rate<32, false, true>() | rate<64, false, true>() | rate<128, false, true>() | rate<32, true, true>() |
         rate<64, true, true>() | rate<128, true, true>();
}
