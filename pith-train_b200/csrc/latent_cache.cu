// Writing the MLA latent cache and reading rows back.
//
// Write, per token:  c = x * rsqrt(mean(x^2) + eps) * w   (512 values),
//   r[j] = p[2j] cos[j] - p[2j+1] sin[j],  r[32+j] = p[2j+1] cos[32+j] + p[2j] sin[32+j]   (64 values, j < 32),
// stored at the token's slot as bf16, or c as e4m3 with one power-of-two factor 2^k a row, k the least integer with
// max|c| <= 448 * 2^k: the division is exact, so the only rounding is e4m3's, and the row read back is exact in bf16.
// One warp per token: a lane holds 16 of the 512 values (two 16-byte loads, 512 contiguous bytes a warp instruction), the
// row sum and maximum are five shuffles each, and every lane rotates one pair of inputs into outputs j and 32 + j. Loads of a
// token are issued before the first use; the kernels are bound by HBM at prompt sizes and by the launch at decode sizes.
// Measured: 64 tokens 2.0 us; 8191 tokens into an 8-bit cache and back out of it 13 us, into a bf16 one 7.7 us (one token a warp,
// so that two dependent loads and the launch are most of it); 32768 rows of a bf16 cache 12.6 us = 6.0 TB/s, 0.93 of the
// measured copy rate.
#include "../../include/pith_b200.h"
#include "common.cuh"
#include "host_common.h"

namespace pith {

constexpr int kLatent = 512, kRope = 64;

struct LatentPlanes {
  void* latent;
  void* rope;
  float* scale;
  FastDiv by_page;
  int64_t slots;  // pages * page_size
  int64_t ls[2], rs[2], ss[2];
};

struct LatentWriteParams {
  LatentPlanes c;
  const __nv_bfloat16* kv;
  const __nv_bfloat16* pe;
  const void* w;
  const void* cos;
  const void* sin;
  const int64_t* slots;
  const int64_t* pos;
  uint32_t* status;
  int64_t n, table_rows;
  FastDiv by_s;
  float eps;
  int64_t kvs[2], ps[2], cs[2], sls[2], pos_s[2];
};

struct LatentReadParams {
  LatentPlanes c;
  const int64_t* slots;
  __nv_bfloat16* latent;
  __nv_bfloat16* pe;
  uint32_t* status;
  int64_t n;
};

__device__ __forceinline__ void bf16x8(uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack_bf16x8(const float* f) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
template <bool F32>
__device__ __forceinline__ void load_f4(const void* base, int64_t off, float* f) {
  if (F32) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + off));
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + off));
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
}
template <bool F32>
__device__ __forceinline__ float load_f(const void* base, int64_t off) {
  if (F32) return __ldg(static_cast<const float*>(base) + off);
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(base) + off));
}
__device__ __forceinline__ void report_index(uint32_t* status, uint32_t what) {
  if (status != nullptr) atomicCAS(status, 0u, (kErrIndex << 24) | what);
}
__device__ __forceinline__ uint32_t pack_e4m3x4(const float* f) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(f[1]), "f"(f[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(f[3]), "f"(f[2]));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
__device__ __forceinline__ void unpack_e4m3x4(uint32_t v, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(v >> (16 * i))));
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
        : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "r"(h2));
  }
}

// 48 registers: five CTAs an SM, so that 8191 tokens are 1.4 waves (with 16 weights and a whole rotation a lane
// held from the start 73, and 7.2 instead of 6.3 us).
template <bool FP8, bool CS32, bool W32>
__global__ void __launch_bounds__(256, 5) latent_write_kernel(const LatentWriteParams p) {
  const int lane = threadIdx.x & 31;
  // One value for the warp, whose lanes reduce a row together: another stream may record an error at any time.
  const uint32_t failed =
      __shfl_sync(0xFFFFFFFFu, p.status != nullptr ? *reinterpret_cast<volatile uint32_t*>(p.status) : 0u, 0);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); t < p.n;
       t += static_cast<int64_t>(gridDim.x) * 8) {
    const int b = p.by_s(static_cast<int>(t)), s = static_cast<int>(t) - b * p.by_s.d;
    // everything that does not depend on another load is requested first
    const int64_t slot = __ldg(p.slots + b * p.sls[0] + s * p.sls[1]);
    int64_t row = 0;
    if (p.pos != nullptr) row = __ldg(p.pos + b * p.pos_s[0] + s * p.pos_s[1]);
    const uint4* x = reinterpret_cast<const uint4*>(p.kv + b * p.kvs[0] + s * p.kvs[1]);
    const uint4 x0 = __ldg(x + lane), x1 = __ldg(x + 32 + lane);
    const uint32_t pe = __ldg(reinterpret_cast<const uint32_t*>(p.pe + b * p.ps[0] + s * p.ps[1]) + lane);
    if (slot < 0 || failed != 0u) continue;  // padding
    if (slot >= p.c.slots || (p.pos != nullptr && (row < 0 || row >= p.table_rows))) {
      if (lane == 0) report_index(p.status, slot >= p.c.slots ? kIdxSlot : kIdxPosition);
      continue;
    }
    const int64_t cs = p.pos != nullptr ? row * p.cs[1] : b * p.cs[0] + s * p.cs[1];
    const float cl = load_f<CS32>(p.cos, cs + lane), ch = load_f<CS32>(p.cos, cs + 32 + lane);
    const float sl = load_f<CS32>(p.sin, cs + lane), sh = load_f<CS32>(p.sin, cs + 32 + lane);
    float f[16];
    bf16x8(x0, f);
    bf16x8(x1, f + 8);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = fmaf(f[i], f[i], sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const float r = rsqrtf(sum * (1.f / kLatent) + p.eps);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {  // the weights are in L1 after the first token: held from the start they cost residency
      float w[4];
      load_f4<W32>(p.w, (i >> 3) * 256 + lane * 8 + (i & 4), w);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[i + j] = f[i + j] * r * w[j];
    }
    const int page = p.c.by_page(static_cast<int>(slot)), in_page = static_cast<int>(slot) - page * p.c.by_page.d;
    const int64_t dst = page * p.c.ls[0] + in_page * p.c.ls[1];
    if (FP8) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(f[i]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      // top = (1 + m / 2^23) 2^e and 448 = 1.75 * 2^8: k = e - 8, or e - 7 where the mantissa is above 1.75
      const uint32_t bits = __float_as_uint(top);
      int k = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7FFFFFu) > 0x600000u ? 7 : 8);
      k = top == 0.f ? 0 : max(k, -100);
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
      float scale = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
      if (bits >= 0x7F800000u) scale = __uint_as_float(0x7FC00000u);  // an infinite value makes the row NaN
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] *= inv;
      uint8_t* d = static_cast<uint8_t*>(p.c.latent) + dst;
      *reinterpret_cast<uint2*>(d + lane * 8) = make_uint2(pack_e4m3x4(f), pack_e4m3x4(f + 4));
      *reinterpret_cast<uint2*>(d + 256 + lane * 8) = make_uint2(pack_e4m3x4(f + 8), pack_e4m3x4(f + 12));
      if (lane == 0) p.c.scale[page * p.c.ss[0] + in_page * p.c.ss[1]] = scale;
    } else {
      uint4* d = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.c.latent) + dst);
      d[lane] = pack_bf16x8(f);
      d[32 + lane] = pack_bf16x8(f + 8);
    }
    const float even = __uint_as_float(pe << 16), odd = __uint_as_float(pe & 0xFFFF0000u);
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.c.rope) + page * p.c.rs[0] + in_page * p.c.rs[1];
    d[lane] = __float2bfloat16_rn(even * cl - odd * sl);
    d[32 + lane] = __float2bfloat16_rn(odd * ch + even * sh);
  }
}

template <bool FP8>
__global__ void __launch_bounds__(256, 8) latent_read_kernel(const LatentReadParams p) {
  const int lane = threadIdx.x & 31;
  const uint32_t failed = p.status != nullptr ? *reinterpret_cast<volatile uint32_t*>(p.status) : 0u;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); t < p.n;
       t += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t slot = __ldg(p.slots + t);
    if (failed != 0u) continue;
    uint4 a = make_uint4(0, 0, 0, 0), b = a, r = a;
    if (slot >= p.c.slots) {
      if (lane == 0) report_index(p.status, kIdxSlot);
    } else if (slot >= 0) {
      const int page = p.c.by_page(static_cast<int>(slot)), in_page = static_cast<int>(slot) - page * p.c.by_page.d;
      const int64_t src = page * p.c.ls[0] + in_page * p.c.ls[1];
      if (lane < 8)
        r = *(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.c.rope) + page * p.c.rs[0] +
                                             in_page * p.c.rs[1]) + lane);
      if (FP8) {
        const uint4 v = *(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.c.latent) + src) + lane);
        const float scale = p.c.scale[page * p.c.ss[0] + in_page * p.c.ss[1]];
        float f[16];
        unpack_e4m3x4(v.x, f);
        unpack_e4m3x4(v.y, f + 4);
        unpack_e4m3x4(v.z, f + 8);
        unpack_e4m3x4(v.w, f + 12);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] *= scale;
        a = pack_bf16x8(f);
        b = pack_bf16x8(f + 8);
      } else {
        const uint4* x = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.c.latent) + src);
        a = x[lane];
        b = x[32 + lane];
      }
    }
    uint4* d = reinterpret_cast<uint4*>(p.latent + t * kLatent);
    if (FP8) {  // a lane holds 16 consecutive values
      d[2 * lane] = a;
      d[2 * lane + 1] = b;
    } else {
      d[lane] = a;
      d[32 + lane] = b;
    }
    if (lane < 8) *(reinterpret_cast<uint4*>(p.pe + t * kRope) + lane) = r;
  }
}

int check_latent_cache(const pith_latent_cache& c) {
  PITH_REQUIRE(c.dtype == PITH_DTYPE_BF16 || c.dtype == PITH_DTYPE_E4M3, "cache dtype must be bf16 or e4m3");
  PITH_REQUIRE(c.pages > 0 && (c.page_size == 16 || c.page_size == 32 || (c.page_size > 0 && c.page_size % 64 == 0)),
               "page_size must be 16, 32 or a multiple of 64 (got %d pages of %d)", c.pages, c.page_size);
  PITH_REQUIRE(c.latent && c.rope && (c.dtype == PITH_DTYPE_BF16 || c.scale), "null cache plane");
  PITH_REQUIRE(static_cast<int64_t>(c.pages) * c.page_size < 2147483648ll, "a cache holds at most 2^31 - 1 rows");
  const int eb = c.dtype == PITH_DTYPE_BF16 ? 2 : 1;
  const int64_t ls0 = axis_stride(c.pages, c.latent_stride[0], 16), rs0 = axis_stride(c.pages, c.rope_stride[0], 16);
  PITH_REQUIRE(aligned16(c.latent) && aligned16(c.rope) && (ls0 * eb) % 16 == 0 && (c.latent_stride[1] * eb) % 16 == 0 &&
                   rs0 % 8 == 0 && c.rope_stride[1] % 8 == 0,
               "cache planes must be 16-byte aligned with 16-byte-multiple strides");
  PITH_REQUIRE(ls0 > 0 && c.latent_stride[1] >= kLatent && rs0 > 0 && c.rope_stride[1] >= kRope, "cache rows overlap");
  return kOk;
}

static LatentPlanes planes_of(const pith_latent_cache& c) {
  LatentPlanes l;
  l.latent = c.latent; l.rope = c.rope; l.scale = c.scale;
  l.by_page = FastDiv(c.page_size);
  l.slots = static_cast<int64_t>(c.pages) * c.page_size;
  for (int i = 0; i < 2; ++i) { l.ls[i] = c.latent_stride[i]; l.rs[i] = c.rope_stride[i]; l.ss[i] = c.scale_stride[i]; }
  return l;
}

// 8 tokens per CTA and pass, at most 8 CTAs per SM (2048 threads)
static int token_grid(int64_t n, unsigned* grid) {
  int dev = 0, sms = 148;
  PITH_CUDA(cudaGetDevice(&dev));
  PITH_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int64_t need = (n + 7) / 8, most = static_cast<int64_t>(sms) * 8;
  *grid = static_cast<unsigned>(need < most ? need : most);
  return kOk;
}

}  // namespace pith

using namespace pith;

extern "C" int pith_latent_write(const pith_latent_write_args* a, void* stream) {
  PITH_REQUIRE(a != nullptr, "null args");
  PITH_REQUIRE(a->B >= 0 && a->S >= 0, "negative size");
  if (int rc = check_latent_cache(a->cache)) return rc;
  if (a->B == 0 || a->S == 0) return kOk;
  PITH_REQUIRE(a->compressed_kv && a->k_pe && a->norm_weight && a->cos && a->sin && a->slots, "null tensor pointer");
  LatentWriteParams p;
  const int64_t sizes[2] = {a->B, a->S};
  for (int i = 0; i < 2; ++i) {
    p.kvs[i] = axis_stride(sizes[i], a->kv_stride[i]);
    p.ps[i] = axis_stride(sizes[i], a->k_pe_stride[i]);
    p.cs[i] = a->cs_stride[i];
    p.sls[i] = a->slots_stride[i];
    p.pos_s[i] = a->positions_stride[i];
  }
  PITH_REQUIRE(aligned16(a->compressed_kv) && aligned16(a->k_pe) && aligned16(a->norm_weight) && aligned16(a->cos) &&
                   aligned16(a->sin) && p.kvs[0] % 8 == 0 && p.kvs[1] % 8 == 0 && p.ps[0] % 8 == 0 && p.ps[1] % 8 == 0 &&
                   p.cs[0] % 4 == 0 && p.cs[1] % 4 == 0,
               "inputs must be 16-byte aligned with strides that are multiples of 8 elements (cos / sin: 4)");
  PITH_REQUIRE((a->cs_dtype == PITH_DTYPE_BF16 || a->cs_dtype == PITH_DTYPE_F32) &&
                   (a->weight_dtype == PITH_DTYPE_BF16 || a->weight_dtype == PITH_DTYPE_F32),
               "norm_weight and cos / sin must be bf16 or fp32");
  PITH_REQUIRE(a->eps >= 0.f, "eps must not be negative");
  if (int rc = require_sm100()) return rc;
  p.c = planes_of(a->cache);
  p.kv = static_cast<const __nv_bfloat16*>(a->compressed_kv);
  p.pe = static_cast<const __nv_bfloat16*>(a->k_pe);
  p.w = a->norm_weight; p.cos = a->cos; p.sin = a->sin;
  p.slots = a->slots; p.pos = a->positions; p.status = a->status;
  p.n = static_cast<int64_t>(a->B) * a->S;
  PITH_REQUIRE(p.n < 2147483648ll, "too many tokens for one call");
  p.by_s = FastDiv(a->S); p.table_rows = a->table_rows; p.eps = a->eps;
  unsigned grid = 1;
  if (int rc = token_grid(p.n, &grid)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fp8 = a->cache.dtype == PITH_DTYPE_E4M3, cs = a->cs_dtype == PITH_DTYPE_F32,
             w = a->weight_dtype == PITH_DTYPE_F32;
  auto kern = fp8 ? (cs ? (w ? latent_write_kernel<true, true, true> : latent_write_kernel<true, true, false>)
                        : (w ? latent_write_kernel<true, false, true> : latent_write_kernel<true, false, false>))
                  : (cs ? (w ? latent_write_kernel<false, true, true> : latent_write_kernel<false, true, false>)
                        : (w ? latent_write_kernel<false, false, true> : latent_write_kernel<false, false, false>));
  kern<<<grid, 256, 0, st>>>(p);
  PITH_CUDA(cudaGetLastError());
  return kOk;
}

extern "C" int pith_latent_read(const pith_latent_read_args* a, void* stream) {
  PITH_REQUIRE(a != nullptr, "null args");
  PITH_REQUIRE(a->n >= 0, "negative size");
  if (int rc = check_latent_cache(a->cache)) return rc;
  if (a->n == 0) return kOk;
  PITH_REQUIRE(a->slots && a->latent && a->k_pe, "null tensor pointer");
  PITH_REQUIRE(aligned16(a->latent) && aligned16(a->k_pe), "outputs must be 16-byte aligned");
  if (int rc = require_sm100()) return rc;
  LatentReadParams p;
  p.c = planes_of(a->cache);
  p.slots = a->slots;
  p.latent = static_cast<__nv_bfloat16*>(a->latent);
  p.pe = static_cast<__nv_bfloat16*>(a->k_pe);
  p.status = a->status; p.n = a->n;
  unsigned grid = 1;
  if (int rc = token_grid(p.n, &grid)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->cache.dtype == PITH_DTYPE_E4M3) latent_read_kernel<true><<<grid, 256, 0, st>>>(p);
  else latent_read_kernel<false><<<grid, 256, 0, st>>>(p);
  PITH_CUDA(cudaGetLastError());
  return kOk;
}
