// The two projections around latent attention, per head h with W = kv_b_proj.weight [H * 256][512]:
//
//   query:   out[t][h][0:512]   = q[t][h][0:128] W[h*256 : h*256+128, :]      (K = 128, N = 512)
//            out[t][h][512:576] = rotary embedding of q[t][h][128:192]
//   output:  out[t][h][v]       = sum_r a[t][h][r] W[h*256+128+v, r]          (K = 512, N = 128)
//
// W is used as the layer holds it: the query's B operand is read MN-major, the output's K-major; tcgen05 with accumulators in
// TMEM, results stored by TMA, which clips the rows behind the last token. A row moves 1.5 KB (query) or 1.3 KB (output) for
// 131 kFLOP: HBM bounds both at prompt sizes, latency at decode sizes, where narrow tiles spread the reading of W over more
// CTAs (a kernel of one tile per CTA). Measured, 16 heads: 32 tokens 3.5 us (query) and 4.5 us (output); 4095 tokens 22.3 us
// = 4.6 TB/s (0.71 of the measured copy rate) and 18.5 us = 4.7 TB/s (0.72), of which the launch, W and the first tile
// take about 4 us.
#include "../../include/pith_b200.h"
#include "common.cuh"
#include "host_common.h"

namespace pith {

struct LatProjParams {
  const __nv_bfloat16* q;  // query only: rope parts
  __nv_bfloat16* out;
  const void* cos;
  const void* sin;
  const int64_t* pos;
  uint32_t* status;
  int H, rows;              // rows of the flattened (or per-batch) token axis
  FastDiv by_s;             // tokens per sequence of the caller's view
  int cs_f32;
  int64_t table_rows;
  int64_t qs[3], cs[2], pos_s[2];
};

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* smem_src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All but the N newest groups of stores have read their shared memory.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void lat_load4(const void* base, int f32, int64_t off, float* f) {
  if (f32) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + off));
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + off));
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
}

// Rotary parts of PASSES x 16 query rows by 128 threads: lane l8 of eight turns inputs [8 l8, 8 l8 + 8) of a row into outputs
// [4 l8, +4) and [32 + 4 l8, +4). All positions, then all other loads are issued before the first use: one after the other
// they took longer than the tile's GEMM.
template <int PASSES>
__device__ __forceinline__ void lat_rope_rows(const LatProjParams& p, int64_t g0, int rows, int h, int t) {
  const int l8 = t & 7;
  int64_t cs[PASSES], from[PASSES];
  bool ok[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    ok[i] = i * 16 + (t >> 3) < rows;
    const int64_t g = g0 + (ok[i] ? i * 16 + (t >> 3) : 0);
    const int b = p.by_s(static_cast<int>(g)), s = static_cast<int>(g) - b * p.by_s.d;
    from[i] = b * p.qs[0] + s * p.qs[1] + h * p.qs[2] + 128;
    cs[i] = b * p.cs[0] + s * p.cs[1];
    if (p.pos != nullptr) {
      const int64_t row = __ldg(p.pos + b * p.pos_s[0] + s * p.pos_s[1]);
      const bool in = row >= 0 && row < p.table_rows;
      if (!in && p.status != nullptr) atomicCAS(p.status, 0u, (kErrIndex << 24) | kIdxPosition);
      ok[i] = ok[i] && in;
      cs[i] = in ? row * p.cs[1] : 0;
    }
  }
  float cl[PASSES][4], ch[PASSES][4], sl[PASSES][4], sh[PASSES][4];
  uint4 x[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (!ok[i]) continue;
    lat_load4(p.cos, p.cs_f32, cs[i] + 4 * l8, cl[i]);
    lat_load4(p.cos, p.cs_f32, cs[i] + 32 + 4 * l8, ch[i]);
    lat_load4(p.sin, p.cs_f32, cs[i] + 4 * l8, sl[i]);
    lat_load4(p.sin, p.cs_f32, cs[i] + 32 + 4 * l8, sh[i]);
    x[i] = __ldg(reinterpret_cast<const uint4*>(p.q + from[i]) + l8);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (!ok[i]) continue;
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float even = __uint_as_float(w[j] << 16), odd = __uint_as_float(w[j] & 0xFFFF0000u);
      lo[j] = even * cl[i][j] - odd * sl[i][j];
      hi[j] = odd * ch[i][j] + even * sh[i][j];
    }
    __nv_bfloat16* d = p.out + ((g0 + i * 16 + (t >> 3)) * p.H + h) * 576 + 512;
    *reinterpret_cast<uint2*>(d + 4 * l8) = make_uint2(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]));
    *reinterpret_cast<uint2*>(d + 32 + 4 * l8) = make_uint2(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]));
  }
}

// Rotary parts of tokens [g0, g1) for all heads, by 256 threads: eight lanes take a token, read its row of the tables once
// and walk its heads sixteen at a time. Beside the GEMM's traffic a dependent load takes microseconds, so that a token's
// position and queries are requested together, then its tables, and one pass of 32 tokens covers a CTA's share of a chunk.
__device__ __forceinline__ void lat_rope_tokens(const LatProjParams& p, int64_t g0, int64_t g1, int t) {
  const int l8 = t & 7;
  constexpr int kHeads = 16;
  for (int64_t g = g0 + (t >> 3); g < g1; g += 32) {
    const int b = p.by_s(static_cast<int>(g)), s = static_cast<int>(g) - b * p.by_s.d;
    int64_t row = 0, cs = b * p.cs[0] + s * p.cs[1];
    if (p.pos != nullptr) row = __ldg(p.pos + b * p.pos_s[0] + s * p.pos_s[1]);
    const __nv_bfloat16* src = p.q + b * p.qs[0] + s * p.qs[1] + 128;
    __nv_bfloat16* dst = p.out + g * p.H * 576 + 512;
    float cl[4], ch[4], sl[4], sh[4];
    for (int h0 = 0; h0 < p.H; h0 += kHeads) {
      uint4 x[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        x[i] = __ldg(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(min(h0 + i, p.H - 1)) * p.qs[2]) + l8);
      if (h0 == 0) {
        if (p.pos != nullptr) {
          if (row < 0 || row >= p.table_rows) {
            if (p.status != nullptr) atomicCAS(p.status, 0u, (kErrIndex << 24) | kIdxPosition);
            break;
          }
          cs = row * p.cs[1];
        }
        lat_load4(p.cos, p.cs_f32, cs + 4 * l8, cl);
        lat_load4(p.cos, p.cs_f32, cs + 32 + 4 * l8, ch);
        lat_load4(p.sin, p.cs_f32, cs + 4 * l8, sl);
        lat_load4(p.sin, p.cs_f32, cs + 32 + 4 * l8, sh);
      }
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (h0 + i >= p.H) break;
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        float lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float even = __uint_as_float(w[j] << 16), odd = __uint_as_float(w[j] & 0xFFFF0000u);
          lo[j] = even * cl[j] - odd * sl[j];
          hi[j] = odd * ch[j] + even * sh[j];
        }
        __nv_bfloat16* d = dst + static_cast<int64_t>(h0 + i) * 576;
        *reinterpret_cast<uint2*>(d + 4 * l8) = make_uint2(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]));
        *reinterpret_cast<uint2*>(d + 32 + 4 * l8) = make_uint2(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]));
      }
    }
  }
}

// A [128 tokens x K] K-major, B [NT columns x K] (query: MN-major), K in blocks of 64 through ST stages.
template <bool QUERY, int NT, int ST>
struct ProjCfg {
  static constexpr int KB = QUERY ? 2 : 8;             // K blocks of 64
  static constexpr int kA = 128 * 128;                 // bytes of an A block
  static constexpr int kB = NT * 128;                  // bytes of a B block
  static constexpr int kStage = kA + kB;
  static constexpr int kOut = NT * 256;                // staged result
  static constexpr int kTiles = ST * kStage > kOut ? ST * kStage : kOut;
  static constexpr int kBars = 2 * ST + 1;
  static constexpr int kAlloc = kTiles + kBars * 8 + 16;
  static constexpr int kCols = NT < 32 ? 32 : NT;
  static constexpr int kThreads = QUERY ? 256 : 128;   // warps 4-7 of the query kernel: rotary parts
};

template <bool QUERY, int NT, int ST>
__global__ void __launch_bounds__(ProjCfg<QUERY, NT, ST>::kThreads)
    latent_proj_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ CUtensorMap tm_out, const LatProjParams p) {
  using L = ProjCfg<QUERY, NT, ST>;
  constexpr int NN = (QUERY ? 512 : 128) / NT;  // column tiles
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kTiles);
  uint64_t* full = bars;
  uint64_t* empty = bars + ST;
  uint64_t* done = bars + 2 * ST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kBars);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AbortCtl ctl{p.status, abort_flag};
  const int nt = blockIdx.x % NN, m0 = (blockIdx.x / NN) * 128, h = blockIdx.y, b = blockIdx.z;

  if (threadIdx.x == 0) {
    *abort_flag = (p.status != nullptr && *reinterpret_cast<volatile uint32_t*>(p.status) != 0u) ? 1u : 0u;
    for (int i = 0; i < ST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(done, 1);
    mbar_fence_init();
    if ((smem_u32(smem) & 1023u) != 0u) report_error(ctl, kErrSmemAlign, smem_u32(smem));
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const bool healthy = *abort_flag == 0u;

  if (healthy) {
    if (warp == 0 && lane == 0) {
      for (int k = 0; k < L::KB; ++k) {
        const int s = k % ST;
        mbar_wait(&empty[s], ((k / ST) & 1) ^ 1, ctl, 0x100 + s);
        uint8_t* st = smem + s * L::kStage;
        mbar_arrive_expect_tx(&full[s], L::kStage);
        tma_load_4d(st, &tm_a, &full[s], k * 64, h, m0, b);
        if (QUERY) {  // 64 rows of W (the K block) x NT columns, as [64 rows][64 columns] blocks
#pragma unroll
          for (int i = 0; i < NT / 64; ++i)
            tma_load_4d(st + L::kA + i * 8192, &tm_w, &full[s], nt * NT + i * 64, 0, h * 256 + k * 64, 0);
        } else {  // NT rows of W x 64 columns (the K block)
          tma_load_4d(st + L::kA, &tm_w, &full[s], k * 64, 0, h * 256 + 128 + nt * NT, 0);
        }
      }
    }
    __syncwarp();
    if (warp == 1) {
      const bool leader = elect_one();
      constexpr uint32_t idesc = make_idesc_bf16(128, NT, false, QUERY);
      for (int k = 0; k < L::KB; ++k) {
        const int s = k % ST;
        mbar_wait(&full[s], (k / ST) & 1, ctl, 0x400 + s);
        tc_fence_after_sync();
        if (leader) {
          const uint64_t ad = make_smem_desc(smem_u32(smem) + s * L::kStage, 16, 1024);
          const uint64_t bd = make_smem_desc(smem_u32(smem) + s * L::kStage + L::kA, QUERY ? 8192 : 16, 1024);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            umma_ss(tmem, desc_advance(ad, i * 32), desc_advance(bd, QUERY ? i * 2048 : i * 32), idesc,
                    (k > 0 || i > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
          if (k + 1 == L::KB) umma_commit(done);
        }
      }
    }
    __syncwarp();
    if (QUERY && warp >= 4) {  // this column tile's share of the rotary parts
      constexpr int RR = 128 / NN;
      const int first = m0 + nt * RR;
      if (first < p.rows)
        lat_rope_rows<(RR + 15) / 16>(p, static_cast<int64_t>(b) * p.rows + first, min(RR, p.rows - first), h,
                                      static_cast<int>(threadIdx.x) - 128);
    } else {
      mbar_wait(done, 0, ctl, 0x800);
      tc_fence_after_sync();
      const int t = threadIdx.x;
      const uint32_t tl = tmem + (static_cast<uint32_t>(warp << 5) << 16);
#pragma unroll
      for (int c = 0; c < NT / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(tl + c * 32, r);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t* v = r + 8 * i;
          const uint4 y = make_uint4(pack_bf16(__uint_as_float(v[0]), __uint_as_float(v[1])),
                                     pack_bf16(__uint_as_float(v[2]), __uint_as_float(v[3])),
                                     pack_bf16(__uint_as_float(v[4]), __uint_as_float(v[5])),
                                     pack_bf16(__uint_as_float(v[6]), __uint_as_float(v[7])));
          if (NT >= 64) {
            const int ch = (c & 1) * 4 + i;
            *reinterpret_cast<uint4*>(smem + (c >> 1) * 16384 + t * 128 + (((ch ^ t) & 7) << 4)) = y;
          } else if (m0 + t < p.rows) {
            *(reinterpret_cast<uint4*>(p.out + ((static_cast<int64_t>(b) * p.rows + m0 + t) * p.H + h) * 128 + nt * NT) + i) = y;
          }
        }
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  if (NT >= 64 && *abort_flag == 0u && threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) tma_store_4d(&tm_out, smem + i * 16384, nt * NT + i * 64, h, m0, b);
    tma_store_commit();
    tma_store_wait_read<0>();  // the shared memory may go once it has been read
  }
  if (*abort_flag != 0u) {  // let copies and MMAs still in flight drain before shared memory and TMEM are handed back
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
  }
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, L::kCols);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Many tokens: a persistent kernel. One CTA per SM takes a contiguous run of (head, column tile, token tile) items with the
// token tile innermost, so that its part of W stays in shared memory (64 KB of the query's, 128 KB of the output's) and only
// the tokens stream: TMA producer (warp 0), MMA issuer (warp 1), epilogue (warps 4-7, two accumulators in TMEM, staged and
// stored by TMA), rotary parts (warps 8-15, query only). One tile per CTA, loads, MMAs and stores one after the other, took
// 28.6 us (query) and 19.2 us (output) for 4095 tokens x 16 heads.
template <bool QUERY>
struct RunCfg {
  static constexpr int NT = QUERY ? 256 : 128;
  static constexpr int NN = QUERY ? 2 : 1;
  static constexpr int KB = QUERY ? 2 : 8;
  static constexpr int kB = NT * 128 * KB;
  static constexpr int ST = QUERY ? 6 : 4;  // 16 KB stages of A
  static constexpr int kAOff = kB;
  static constexpr int kOutOff = kAOff + ST * 16384;
  static constexpr int kBarOff = kOutOff + NT * 256;
  static constexpr int kBars = 2 * ST + 6;
  static constexpr int kAlloc = kBarOff + kBars * 8 + 16;
  static constexpr int kThreads = QUERY ? 512 : 256;
  static_assert(kAlloc <= 232448, "shared memory");
};

template <bool QUERY>
__global__ void __launch_bounds__(RunCfg<QUERY>::kThreads, 1)
    latent_proj_run_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                           const __grid_constant__ CUtensorMap tm_out, const LatProjParams p, int tile, FastDiv by_tiles,
                           FastDiv by_groups, int items, int per_group, int tokens, int token_share) {
  using L = RunCfg<QUERY>;
  constexpr int NT = L::NT, NN = L::NN, KB = L::KB, ST = L::ST;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* full = bars;
  uint64_t* empty = bars + ST;
  uint64_t* b_full = bars + 2 * ST;
  uint64_t* b_empty = b_full + 1;
  uint64_t* acc_full = b_full + 2;   // [2]
  uint64_t* acc_empty = b_full + 4;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kBars);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AbortCtl ctl{p.status, abort_flag};
  // Items i0, i0 + step, ... below i1; item = (group, token tile), group = (batch, head, column tile). With per_group CTAs
  // for each group, neighbouring CTAs take the same token tile of different heads, so that the rows of a token, which lie
  // together, are read and written at about the same time. Otherwise (more groups than CTAs) equal runs of items.
  const int me = blockIdx.x, ctas = gridDim.x;
  int i0, i1, step;
  if (per_group > 0) {
    const int first = by_groups(me), g = me - first * by_groups.d;
    i0 = g * by_tiles.d + first;
    i1 = (g + 1) * by_tiles.d;
    step = per_group;
  } else {
    const int share = items / ctas, more = items - share * ctas;
    i0 = me * share + min(me, more);
    i1 = i0 + share + (me < more ? 1 : 0);
    step = 1;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(b_full, 1);
    mbar_init(b_empty, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 128); }
    mbar_fence_init();
  }
  if (threadIdx.x == 64) {
    *abort_flag = (p.status != nullptr && *reinterpret_cast<volatile uint32_t*>(p.status) != 0u) ? 1u : 0u;
    if ((smem_u32(smem) & 1023u) != 0u) report_error(ctl, kErrSmemAlign, smem_u32(smem));
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * NT);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  if (*abort_flag != 0u) i1 = i0;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t s = 0, ph = 1, bph = 1;
      int group = -1;
      for (int it = i0; it < i1; it += step) {
        const int g = by_tiles(it), m0 = (it - g * by_tiles.d) * tile;
        const int nt = g % NN, h = g / NN % p.H, b = g / NN / p.H;
        if (g != group) {
          group = g;
          mbar_wait(b_empty, bph, ctl, 0x200);
          bph ^= 1;
          mbar_arrive_expect_tx(b_full, L::kB);
          for (int k = 0; k < KB; ++k) {
            if (QUERY) {  // 64 rows of W (the K block) x NT columns, as [64 rows][64 columns] blocks
              for (int i = 0; i < NT / 64; ++i)
                tma_load_4d(smem + k * (NT * 128) + i * 8192, &tm_w, b_full, nt * NT + i * 64, 0, h * 256 + k * 64, 0);
            } else {      // NT rows of W x 64 columns (the K block)
              tma_load_4d(smem + k * (NT * 128), &tm_w, b_full, k * 64, 0, h * 256 + 128, 0);
            }
          }
        }
        for (int k = 0; k < KB; ++k) {
          mbar_wait(&empty[s], ph, ctl, 0x100 + s);
          mbar_arrive_expect_tx(&full[s], tile * 128);
          tma_load_4d(smem + L::kAOff + s * 16384, &tm_a, &full[s], k * 64, h, m0, b);
          if (++s == ST) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t idesc = make_idesc_bf16(128, NT, false, QUERY);
    const uint64_t ad0 = make_smem_desc(smem_u32(smem) + L::kAOff, 16, 1024);
    const uint64_t bd0 = make_smem_desc(smem_u32(smem), QUERY ? 8192 : 16, 1024);
    uint32_t s = 0, ph = 0, bph = 0;
    int group = -1;
    uint32_t n = 0;
    for (int it = i0; it < i1; it += step, ++n) {
      const uint32_t buf = n & 1;
      const int g = by_tiles(it);
      if (g != group) {
        group = g;
        mbar_wait(b_full, bph, ctl, 0x300);
        bph ^= 1;
      }
      mbar_wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1, ctl, 0x500 + buf);
      for (int k = 0; k < KB; ++k) {
        mbar_wait(&full[s], ph, ctl, 0x400 + s);
        tc_fence_after_sync();
        const uint64_t ad = desc_advance(ad0, s * 16384), bd = desc_advance(bd0, k * (NT * 128));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (leader)
            umma_ss(tmem + buf * NT, desc_advance(ad, i * 32), desc_advance(bd, QUERY ? i * 2048 : i * 32), idesc,
                    (k > 0 || i > 0) ? 1u : 0u);
        if (leader) umma_commit(&empty[s]);
        if (++s == ST) { s = 0; ph ^= 1; }
      }
      if (leader) {
        umma_commit(&acc_full[buf]);
        if (it + step < i1 && by_tiles(it + step) != g) umma_commit(b_empty);
      }
    }
  } else if (warp >= 4 && warp < 8) {
    const int t = static_cast<int>(threadIdx.x) & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) << 5) << 16;
    uint8_t* out = smem + L::kOutOff;
    uint32_t n = 0;
    for (int it = i0; it < i1; it += step, ++n) {
      const uint32_t buf = n & 1;
      const int g = by_tiles(it), m0 = (it - g * by_tiles.d) * tile;
      const int nt = g % NN, h = g / NN % p.H, b = g / NN / p.H;
      mbar_wait(&acc_full[buf], (n >> 1) & 1, ctl, 0x800 + buf);
      tc_fence_after_sync();
#pragma unroll 1
      for (int q = 0; q < NT / 64; ++q) {  // 64 columns: staged, and on their way while the next ones are read
        if (t == 0) tma_store_wait_read<NT / 64 - 1>();  // this part's previous contents have been read
        named_bar_sync(1, 128);
        uint8_t* dst = out + q * 16384 + t * 128;
        uint32_t r[64];
        tmem_ld32(tmem + lanes + buf * NT + q * 64, r);
        tmem_ld32(tmem + lanes + buf * NT + q * 64 + 32, r + 32);
        tmem_wait_ld();
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          const uint32_t* v = r + 8 * ch;
          *reinterpret_cast<uint4*>(dst + (((ch ^ t) & 7) << 4)) =
              make_uint4(pack_bf16(__uint_as_float(v[0]), __uint_as_float(v[1])),
                         pack_bf16(__uint_as_float(v[2]), __uint_as_float(v[3])),
                         pack_bf16(__uint_as_float(v[4]), __uint_as_float(v[5])),
                         pack_bf16(__uint_as_float(v[6]), __uint_as_float(v[7])));
        }
        fence_proxy_async_smem();
        named_bar_sync(1, 128);
        if (t == 0 && *abort_flag == 0u) {
          tma_store_4d(&tm_out, out + q * 16384, nt * NT + q * 64, h, m0, b);
          tma_store_commit();
        }
      }
      tc_fence_before_sync();
      mbar_arrive(&acc_empty[buf]);
    }
    if (t == 0) tma_store_wait_read<0>();
  } else if (QUERY && warp >= 8) {
    // an equal share of the tokens, whatever the CTA's items: with the rotary part of its own (head, token) rows every head
    // read the tables again, and the kernel waited for these warps (33.7 us)
    if (*abort_flag == 0u)
      lat_rope_tokens(p, static_cast<int64_t>(me) * token_share, min(tokens, (me + 1) * token_share),
                      static_cast<int>(threadIdx.x) - 256);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 2 * NT);
  }
}

// Tensor maps of W (boxes of 64 columns and `rows` rows) and of the contiguous result (64 columns, `tile` tokens).
template <bool QUERY>
static int proj_maps(const pith_latent_proj_args* a, int64_t B, int64_t S, int rows, int tile, CUtensorMap* tw,
                     CUtensorMap* to) {
  constexpr int kIn = QUERY ? 576 : 128;
  const int64_t ws[3] = {static_cast<int64_t>(a->H) * 256 * a->weight_stride, a->weight_stride, 512};
  if (int rc = make_tensor_map(tw, a->weight, 2, 1, static_cast<int64_t>(a->H) * 256, 1, 512, ws, 64, rows)) return rc;
  const int64_t os[3] = {S * a->H * kIn, static_cast<int64_t>(a->H) * kIn, kIn};
  return make_tensor_map(to, a->out, 2, B, S, a->H, kIn, os, 64, tile);
}

template <bool QUERY>
static int launch_proj_run(const pith_latent_proj_args* a, const LatProjParams& p, int64_t B, int64_t S, const int64_t xs[3],
                           int sms, cudaStream_t st) {
  using L = RunCfg<QUERY>;
  const int64_t groups = B * a->H * L::NN;
  const int per_group = groups <= sms ? static_cast<int>(sms / groups) : 0;
  // Tokens per tile, 64 to 128: what the CTA with the most tiles has to stream decides (4095 tokens, nine CTAs a head: 36
  // tiles of 114 are four rounds, 32 of 128 are also four). A tile costs about 8 tokens of its own.
  int tile = 128;
  int64_t best = -1;
  for (int r = 128; r >= 64; r -= 2) {
    const int64_t mt = (S + r - 1) / r;
    const int64_t rounds = per_group > 0 ? (mt + per_group - 1) / per_group : (mt * groups + sms - 1) / sms;
    if (best < 0 || rounds * (r + 8) < best) {
      best = rounds * (r + 8);
      tile = r;
    }
  }
  CUtensorMap ta, tw, to;
  if (int rc = make_tensor_map(&ta, a->x, 2, B, S, a->H, QUERY ? 192 : 512, xs, 64, tile)) return rc;
  if (int rc = proj_maps<QUERY>(a, B, S, QUERY ? 64 : L::NT, tile, &tw, &to)) return rc;
  auto kern = latent_proj_run_kernel<QUERY>;
  PITH_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc));
  const int64_t mt = (S + tile - 1) / tile, items = mt * groups;
  PITH_REQUIRE(items < 2147483647 - 1024, "too many tokens, heads or sequences");
  const int64_t ctas = per_group > 0 ? groups * per_group : items < sms ? items : sms;
  kern<<<static_cast<unsigned>(ctas), L::kThreads, L::kAlloc, st>>>(
      ta, tw, to, p, tile, FastDiv(static_cast<int>(mt)), FastDiv(static_cast<int>(groups)), static_cast<int>(items), per_group,
      static_cast<int>(B * S), static_cast<int>((B * S + ctas - 1) / ctas));
  PITH_CUDA(cudaGetLastError());
  return kOk;
}

template <bool QUERY, int NT, int ST>
static int launch_proj(const pith_latent_proj_args* a, const LatProjParams& p, int64_t B, int64_t S, const int64_t xs[3],
                       cudaStream_t st) {
  using L = ProjCfg<QUERY, NT, ST>;
  constexpr int NN = (QUERY ? 512 : 128) / NT;
  CUtensorMap ta, tw, to;
  if (int rc = make_tensor_map(&ta, a->x, 2, B, S, a->H, QUERY ? 192 : 512, xs, 64, 128)) return rc;
  if (int rc = proj_maps<QUERY>(a, B, S, QUERY ? 64 : NT, 128, &tw, &to)) return rc;
  auto kern = latent_proj_kernel<QUERY, NT, ST>;
  PITH_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc));
  const int64_t mt = (S + 127) / 128;
  PITH_REQUIRE(mt * NN < 2147483647 && a->H <= 65535 && B <= 65535, "too many tokens, heads or sequences");
  kern<<<dim3(static_cast<unsigned>(mt * NN), a->H, static_cast<unsigned>(B)), L::kThreads, L::kAlloc, st>>>(ta, tw, to, p);
  PITH_CUDA(cudaGetLastError());
  return kOk;
}

template <bool QUERY>
static int latent_proj(const pith_latent_proj_args* a, void* stream) {
  PITH_REQUIRE(a != nullptr, "null args");
  PITH_REQUIRE(a->B >= 0 && a->S >= 0 && a->H >= 0, "negative size");
  if (a->B == 0 || a->S == 0 || a->H == 0) return kOk;
  PITH_REQUIRE(a->x && a->weight && a->out, "null tensor pointer");
  PITH_REQUIRE(aligned16(a->out), "out must be 16-byte aligned");
  LatProjParams p = {};
  p.qs[0] = axis_stride(a->B, a->x_stride[0]);
  p.qs[1] = axis_stride(a->S, a->x_stride[1]);
  p.qs[2] = axis_stride(a->H, a->x_stride[2]);
  if (QUERY) {
    PITH_REQUIRE(a->cos && a->sin, "null tensor pointer");
    PITH_REQUIRE(aligned16(a->cos) && aligned16(a->sin) && a->cs_stride[0] % 4 == 0 && a->cs_stride[1] % 4 == 0,
                 "cos / sin must be 16-byte aligned with strides that are multiples of 4 elements");
    PITH_REQUIRE(a->cs_dtype == PITH_DTYPE_BF16 || a->cs_dtype == PITH_DTYPE_F32, "cos / sin must be bf16 or fp32");
  }
  PITH_REQUIRE(aligned16(a->x) && p.qs[0] % 8 == 0 && p.qs[1] % 8 == 0 && p.qs[2] % 8 == 0,
               "%s must be 16-byte aligned with strides that are multiples of 8 elements", QUERY ? "q" : "attn");
  PITH_REQUIRE((a->B == 1 || p.qs[0] > 0) && (a->S == 1 || p.qs[1] > 0) && (a->H == 1 || p.qs[2] > 0),
               "%s must not repeat elements (an expanded view)", QUERY ? "q" : "attn");
  PITH_REQUIRE(aligned16(a->weight) && a->weight_stride > 0 && a->weight_stride % 8 == 0,
               "kv_b_weight must be 16-byte aligned with a row stride that is a multiple of 8 elements");
  PITH_REQUIRE(static_cast<int64_t>(a->B) * a->S < 2147483647 - 65536, "too many tokens");
  if (int rc = require_sm100()) return rc;
  // One token axis where the strides allow it: a batch of single tokens fills the tiles. The tensor maps want a stride for
  // axes of one element too.
  int64_t B = a->B, S = a->S;
  int64_t xs[3] = {p.qs[0], p.qs[1], axis_stride(a->H, p.qs[2], QUERY ? 192 : 512)};
  if (S == 1 || B == 1 || xs[0] == S * xs[1]) {
    if (S == 1) xs[1] = xs[0];
    S *= B;
    B = 1;
  }
  xs[1] = axis_stride(S, xs[1], a->H * xs[2]);
  xs[0] = axis_stride(B, xs[0], S * xs[1]);
  p.q = static_cast<const __nv_bfloat16*>(a->x);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.cos = a->cos; p.sin = a->sin; p.pos = a->positions; p.status = a->status;
  p.H = a->H; p.rows = static_cast<int>(S); p.by_s = FastDiv(a->S); p.cs_f32 = a->cs_dtype == PITH_DTYPE_F32;
  p.table_rows = a->table_rows;
  for (int i = 0; i < 2; ++i) { p.cs[i] = a->cs_stride[i]; p.pos_s[i] = a->positions_stride[i]; }
  int dev = 0, sms = 148;
  PITH_CUDA(cudaGetDevice(&dev));
  PITH_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t tiles = (S + 127) / 128 * B * a->H;
  // narrow tiles while the wide ones would leave SMs without a CTA
  if constexpr (QUERY) {
    if (tiles * 2 < sms) return launch_proj<true, 64, 2>(a, p, B, S, xs, st);
    return launch_proj_run<true>(a, p, B, S, xs, sms, st);
  } else {
    if (tiles < sms) return launch_proj<false, 32, 8>(a, p, B, S, xs, st);
    return launch_proj_run<false>(a, p, B, S, xs, sms, st);
  }
}

}  // namespace pith

extern "C" int pith_latent_query(const pith_latent_proj_args* a, void* stream) { return pith::latent_proj<true>(a, stream); }
extern "C" int pith_latent_output(const pith_latent_proj_args* a, void* stream) { return pith::latent_proj<false>(a, stream); }
