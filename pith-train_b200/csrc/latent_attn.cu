// Attention in the absorbed MLA form over a paged latent cache: keys are [c | r] (512 + 64), values are c, shared by all
// heads, so the rows of one sequence are its (new token, head) pairs and all of them read the same keys:
//
//   s[m][n] = scale (q_c[m] . c_n + q_r[m] . r_n),   out[m] = sum_n softmax_n(s[m])[n] c_n,   512 outputs a row.
//
// Decoding has few rows (16 heads) and many keys, so both GEMMs run transposed, with the keys or the output dimensions on
// the 128 lanes of the tensor core and the rows as its N:
//   S^T[128 keys x NT rows] = [c | r]_tile * Q^T         A = cache tile, K-major, as it lies in memory
//   O^T[128 dims x NT rows] += c_tile^T * P^T            A = the same tile read MN-major; four of these make the 512
// A tile of 128 keys is thus read from HBM once, staged once by TMA and used by both. At NT = 16 a tile costs 68 MMAs of
// a narrow N beside the 147 KB (bf16) that HBM delivers to one SM in ~6000 cycles: the kernel is bound by HBM until a
// sequence has more than ~64 rows.
//
// An 8-bit cache stays 8-bit up to the tensor core (kind::f8f6f4). The bf16 query is split into two e4m3 terms
// q 2^-k = hi + lo / 16 (8 significant bits, all that bf16 has, down to 2^-13 of the row's largest element, and 2^-22 of it
// absolutely), the weights likewise, and hi and lo are separate columns of the same MMA: an MMA of 128 x N x 32 bytes costs
// 39.6 cycles at N = 16, 40.6 at 32, 48.7 at 64 (what bounds it is reading A from shared memory; microbench/latent_mma_rate.cu),
// so the second half is nearly free. The row factor of a key enters the score in registers and the weight as w_n = 2^(s_n + log2 scale_n - ref):
// ref is the running maximum of s_n + log2 scale_n (or up to 2^4 below it). The two terms hold weights above 2^-9 of the
// reference to 2^-9 of themselves; below that their steps are 2^-17 of the reference, whatever the weight. Rounded to the
// nearest step, the many small weights behind one large one (a context whose first token outweighs each other one by 2^18)
// would all be lost, or all be up to doubled: 18 % of the output at 99 000 keys. So each key's weights get an offset within half
// a step, taken from the multiples of the golden ratio, before they are rounded: a share of the keys is then rounded up that is
// what the weight is of a step, and sums over keys keep their value. What is left is the scatter of c over the keys that were
// rounded up, at most sqrt(2^-17 W) of it for small weights that add up to W references, against a sum of at least 1 + W:
// below 2^-9 of the result at any number of keys. The row sums take the weights as they were.
// With a bf16 cache the weights are rounded to bf16, 2^-8 of each at most: both operands of that MMA have one type, and a second
// term of 8 more bits would double the columns, which TMEM has not for 64 rows. The results are 0.0019 to 0.0021 of their norm
// from 64 bits; their own rounding is 0.0017.
//
// Work split: the (sequence, row tile, 64 keys) units of the launch form one line which is cut into one equal piece per
// CTA, so any mix of lengths is balanced without a schedule from the host (lengths are read on the device; short sequences
// stay whole, see lat_plan). A piece that covers a row tile completely stores its result; the others store an fp32 partial
// (O, ref, l), at most two per CTA, and the merge kernel adds them in key order.
//
// Roles: warp 0 TMA producer (one lane per page), warp 1 issues the score GEMMs, warp 2 the output GEMMs, warp 3 loads
// queries (with one or three more for NT = 16, and the softmax warps' help for NT = 32, 8-bit), one or two warpgroups softmax
// and epilogue (thread = key, then = output dimension). The running maximum is moved only when a score exceeds the reference by
// more than 2^8 (8-bit: 2^4), decided by one barrier reduction per tile. The score GEMM of the next tile runs under this tile's
// softmax as far as the ring of latent slots holds it: completely with an 8-bit cache, two of four slots at NT = 16, none at
// NT = 64, whose query and tile fill the shared memory.
//
// Measured (16 heads, CUDA events over a captured graph): 64 sequences of 130 to 8191 keys, bf16: 65 us, 4.8 TB/s, 0.74 of
// the measured copy rate; the loop itself streams 6 TB/s, the rest is 3 us until the first load, the pieces' ends and the
// merge. 8 sequences of 9000 to 131071 keys, e4m3: 76 us, 5.5 TB/s, 0.85. Shorter tiles (64 keys, more of the ring in
// flight) were slower: 75 and 122 us. 250 tokens of a prompt over 6001 keys, bf16: 78 us, 650 TFLOP/s, the serial chain score
// GEMM (2.2k cycles) - softmax (1.5k) - output GEMM (1.5k) of a tile; the expanded form is the one for long chunks. 16 trees
// of 13 tokens over 500 to 4097 keys, e4m3: 48 us; a tile takes 2600 cycles (its MMAs 1750), as the slots of the tile after
// the next are free, and loaded, only once this tile's output GEMM has completed, and a piece's begin and end take as long
// as four.
#include "common.cuh"
#include "host_common.h"

namespace pith {

constexpr int kLat = 512, kRp = 64;
constexpr int kTile = 128;  // keys per tile
constexpr int kBox = 64;    // rows of a TMA box at most; work is cut at its multiples
constexpr int kMaxExtra = 8;
// Query rows that the loader converts where the softmax warps do the others: an equal share of a CTA's first query; of later
// ones it may begin before those warps have finished with the piece.
__device__ __forceinline__ int loader_rows(uint32_t loads) { return loads == 0 ? 4 : 8; }
constexpr float kNoRef = -1e30f;  // reference of a row that has seen no key (finite: -inf - ref must stay -inf)
constexpr int kColS = 256, kColR = 384;  // TMEM columns of S^T and of its rope part (8-bit), two of each; O^T starts at 0

template <int NT, bool FP8>
struct LatCfg {
  static constexpr int NC = FP8 ? 2 * NT : NT;           // columns of S^T and O^T
  // Units of 64 keys that beginning another piece costs a CTA: what its epilogue, its query and the empty pipeline take
  // over the time of a unit. About two thirds as much made 16 trees of 13 tokens 3 (bf16) and 6 % (8-bit) slower and nothing
  // faster; half as much again changed most batches by less than 1 % and some by 3 %, either way.
  static constexpr int kExtra = FP8 ? (NT == 16 ? 4 : 8) : (NT == 16 ? 2 : NT == 32 ? 3 : 5);
  static_assert(kExtra <= kMaxExtra, "the host checks the line's length with kMaxExtra");
  static constexpr int G = NT >= 32 ? 2 : 1;             // softmax warpgroups, each with CW of the rows
  static constexpr int CW = NT / G;
  // Query loaders: warp 3, and more behind the softmax warps where the register file has room for them (at most three warps
  // per scheduler).
  static constexpr int kLoadWarps = NT > 16 ? 1 : FP8 ? 4 : 2;
  static constexpr bool kHelp = FP8 && NT == 32;  // the softmax warps convert the rows behind the first eight of a query
  static constexpr int kThreads = 128 + 128 * G + (kLoadWarps - 1) * 32;
  static constexpr int kSlot = FP8 ? 16384 : 32768;      // 128 keys x 128 dims of the latent plane
  static constexpr int kQLat = NT * 1024;                // bf16: 8 blocks [NT][64]; 8-bit: 4 blocks [hi, lo][NT][128]
  static constexpr int kQ = kQLat + NT * 128;
  static constexpr int kP = NT * 256;
  static constexpr int kPRow = NT * 2;                   // bytes of a key's weights: NC columns
  static constexpr int kMisc = NT == 16 ? 1024 : 4096;
  // bf16: P overlays the rope tile, which the score GEMM has finished with when P is written; 8-bit: two buffers
  static constexpr int kFixed = 16384 + kQ + (FP8 ? 2 * kP : 0) + kMisc;
  static constexpr int NS = (232448 - kFixed) / kSlot;
  static constexpr int kScores = NS > 4 ? 2 : 1;  // buffers of S^T: a ring of one tile has no slots for a second
  static constexpr int kRopeOff = NS * kSlot;
  static constexpr int kQOff = kRopeOff + 16384;         // one rope tile, 128 keys x 64 dims
  static constexpr int kPOff = FP8 ? kQOff + kQ : kRopeOff;
  static constexpr int kMiscOff = FP8 ? kPOff + 2 * kP : kQOff + kQ;
  static constexpr int kAlloc = kMiscOff + kMisc;
  static constexpr int kBars = 2 * NS + 10;
  static_assert(NS >= 4, "a tile's four latent slots must fit at once");
  static_assert(!FP8 || (NS >= 9 && NS <= 12), "the 8-bit pipeline holds two tiles, and some");
  static_assert(kBars % 2 == 0 && kBars * 8 + 16 + 48 + NT * 44 <= kMisc, "misc area too small");
  static_assert(kAlloc <= 232448, "shared memory");
  static_assert(4 * NC <= kColS && kColS + 2 * NC <= kColR && kColR + 2 * NT <= 512, "TMEM columns");
};

struct LatAttnParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;  // [B][Sq][H][512] contiguous
  float* lse;          // [B][H][Sq] contiguous, log2 domain, optional
  const int32_t* table;
  const int32_t* lens;
  const int32_t* qlens;
  const uint8_t* tree;
  const float* scale;
  float* part_o;      // [2 G][NT / 4][512][4 columns]
  float2* part_ml;    // [2 G][NT]: reference, sum
  int4* part_info;    // [G]: entry continued from the previous CTA, entry begun and not finished, its slot
  uint32_t* status;
  int B, Sq, H, R, RT, pages, page_size, max_keys;
  int unit_log2;          // keys per unit of work
  int whole;              // a unit is all of an entry
  FastDiv by_h, by_rt, by_page;
  int tile_pages, tile_rows;  // a tile's keys as pages and rows
  float scale_log2;
  int64_t qs[3], table_stride, tree_stride[2], scale_stride[2];
};

// One entry of the work line: row tile rt of sequence b.
struct LatEntry {
  int b, r0, len, nq, keys;  // keys: how many its rows can see at most
};
template <int NT>
__device__ __forceinline__ LatEntry lat_entry(const LatAttnParams& p, int e) {
  LatEntry x;
  x.b = p.by_rt(e);
  x.r0 = (e - x.b * p.RT) * NT;
  x.len = min(max(__ldg(p.lens + x.b), 0), p.max_keys);
  x.nq = p.qlens != nullptr ? min(max(__ldg(p.qlens + x.b), 0), p.Sq) : p.Sq;
  const int last = min(p.by_h(min(x.r0 + NT, p.R) - 1), x.nq - 1);
  x.keys = p.by_h(x.r0) >= x.nq ? 0 : p.tree != nullptr ? x.len : max(min(x.len, x.len - x.nq + last + 1), 0);
  return x;
}
__device__ __forceinline__ int lat_units(const LatAttnParams& p, int keys) {
  return max((keys + (1 << p.unit_log2) - 1) >> p.unit_log2, 1);
}

// Walks the pieces of this CTA's share of the line. Every role keeps its own copy. An entry takes `extra` places of the line
// in front of its units: what beginning another piece costs a CTA.
template <int NT>
struct LatWalk {
  int e, off, left, extra;  // off: place inside entry e
  LatEntry x;
  int k0, k1;   // keys [k0, k1) of the entry
  bool begins, ends;
  __device__ __forceinline__ bool next(const LatAttnParams& p) {
    while (left > 0) {
      x = lat_entry<NT>(p, e);
      const int n = lat_units(p, x.keys) + extra;
      const int take = min(n - off, left), u0 = max(off - extra, 0), u1 = off + take - extra;
      k0 = u0 << p.unit_log2;
      k1 = min(x.keys, u1 << p.unit_log2);
      begins = u0 == 0;
      ends = off + take == n;
      left -= take;
      if (ends) { ++e; off = 0; } else { off += take; }
      if (u1 > u0) return true;  // else the share ends in front of the entry's first unit
    }
    return false;
  }
  __device__ __forceinline__ int tiles() const { return (k1 - k0 + kTile - 1) / kTile; }
};

__device__ __forceinline__ void umma_ss_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor for kind::f8f6f4 with e4m3 inputs (format 0) and fp32 accumulation.
constexpr uint32_t make_idesc_e4m3(int m, int n, bool mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(mn_major) << 15) | (static_cast<uint32_t>(mn_major) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Descriptor of an MN-major operand whose rows are one swizzle atom of 32, 64 or 128 bytes wide.
__device__ __forceinline__ uint64_t make_row_desc(uint32_t smem_addr, int row_bytes) {
  const uint64_t d = make_smem_desc(smem_addr, 16, 8 * row_bytes) & ~(static_cast<uint64_t>(7) << 61);
  return d | (static_cast<uint64_t>(row_bytes == 128 ? 2 : row_bytes == 64 ? 4 : 6) << 61);
}
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t* r) {
  static_assert(N == 16 || N % 32 == 0, "columns");
  if (N == 16) tmem_ld16(addr, r);
#pragma unroll
  for (int i = 0; i < N / 32; ++i) tmem_ld32(addr + 32 * i, r + 32 * i);
}
__device__ __forceinline__ bool named_bar_or(uint32_t id, uint32_t nthreads, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred a, b;\n\t"
      "setp.ne.u32 a, %1, 0;\n\t"
      "bar.red.or.pred b, %2, %3, a;\n\t"
      "selp.u32 %0, 1, 0, b;\n\t"
      "}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred)), "r"(id), "r"(nthreads)
      : "memory");
  return r != 0;
}
// Two floats of at most 448 as e4m3 pairs hi + lo / 16. They pass through fp16 (11 significant bits, and its least step,
// 2^-24, is below everything that lo can hold), where the remainder of the first rounding is exact.
__device__ __forceinline__ void split_e4m3x2(float a, float b, uint16_t& hi, uint16_t& lo) {
  asm("{\n\t.reg .b32 h, r, d, z;\n\t"
      "cvt.rn.f16x2.f32 h, %3, %2;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 %0, h;\n\t"
      "cvt.rn.f16x2.e4m3x2 r, %0;\n\t"
      "sub.rn.f16x2 d, h, r;\n\t"
      "mov.b32 z, 0x4C004C00;\n\t"  // 16, 16
      "mul.rn.f16x2 d, d, z;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 %1, d;\n\t}"
      : "=&h"(hi), "=h"(lo) : "f"(a), "f"(b));
}

// Adds a byte offset to the address field of a descriptor. The address never carries out of the lower word, and said so the
// upper word stays the constant that it is: half the moves in front of every MMA.
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) {
  const uint32_t lo = static_cast<uint32_t>(desc) + (bytes >> 4), hi = static_cast<uint32_t>(desc >> 32);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ void cp_async16(uint32_t smem_dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Reduces N per-lane columns over the 32 lanes: halves of the columns are exchanged for halves of the lanes until a lane
// holds max(N / 32, 1) columns, about N shuffles in all. Afterwards v[i] of a lane is column i + first_column(lane).
template <int N, bool MAX>
__device__ __forceinline__ void reduce_cols(float* v, int lane) {
  int n = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool upper = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const float other = __shfl_xor_sync(0xFFFFFFFFu, upper ? v[i] : v[i + n], o);
          const float own = upper ? v[i + n] : v[i];
          v[i] = MAX ? fmaxf(own, other) : own + other;
        }
      }
    } else {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
      v[0] = MAX ? fmaxf(v[0], other) : v[0] + other;
    }
  }
}
template <int N>
__device__ __forceinline__ int first_column(int lane) {
  int c = 0, n = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (n > 1) {
      n >>= 1;
      if (lane & o) c += n;
    }
  return c;
}

template <int I>
struct Int { static constexpr int value = I; };

// Where the key of one thread stands in the block table, and that of the tiles after it: no division on the way (two took the
// producer 600 cycles a tile, which delayed its loads).
struct LatPage {
  int index, row;  // into the sequence's table; row of that page
  __device__ __forceinline__ LatPage(const LatAttnParams& p, int n) : index(p.by_page(n)), row(n - index * p.page_size) {}
  __device__ __forceinline__ void next_tile(const LatAttnParams& p) {
    index += p.tile_pages;
    row += p.tile_rows;
    if (row >= p.page_size) { row -= p.page_size; ++index; }
  }
};

// Shared-memory scalars behind the tiles.
template <int NT, bool FP8>
struct LatShared {
  using L = LatCfg<NT, FP8>;
  uint8_t* base;
  uint64_t* bars;
  __device__ explicit LatShared(uint8_t* smem) : base(smem), bars(reinterpret_cast<uint64_t*>(smem + L::kMiscOff)) {}
  __device__ uint64_t* full(int i) const { return bars + i; }
  __device__ uint64_t* empty(int i) const { return bars + L::NS + i; }
  __device__ uint64_t* rfull() const { return bars + 2 * L::NS; }
  __device__ uint64_t* rempty() const { return bars + 2 * L::NS + 1; }
  __device__ uint64_t* q_full() const { return bars + L::kBars - 8; }
  __device__ uint64_t* q_empty() const { return bars + L::kBars - 7; }
  __device__ uint64_t* s_full(int i) const { return bars + L::kBars - 6 + i; }
  // One for even and one for odd tiles each: a softmax warpgroup may be a tile ahead of the other, and of the output GEMM.
  __device__ uint64_t* p_full(uint32_t tile) const { return bars + L::kBars - 4 + (tile & 1); }
  __device__ uint64_t* o_full(uint32_t tile) const { return bars + L::kBars - 2 + (tile & 1); }  // its output GEMM is complete
  __device__ uint32_t* tmem_slot() const { return reinterpret_cast<uint32_t*>(bars + L::kBars); }  // [0] base, [1] abort flag
  __device__ int* scan() const { return reinterpret_cast<int*>(bars + L::kBars + 1); }             // [12 warps] + start
  __device__ uint32_t* poisoned() const { return reinterpret_cast<uint32_t*>(scan() + 2); }        // later: a bit per key
  __device__ float* cols() const { return reinterpret_cast<float*>(bars + L::kBars + 8); }         // 11 NT words
  __device__ float* ref() const { return cols(); }
  __device__ float* fac() const { return cols() + NT; }
  __device__ float* qk(int i) const { return cols() + (2 + i) * NT; }
  __device__ float* red(int g) const { return cols() + 4 * NT + g * 4 * L::CW; }  // [4 warps][CW]
  __device__ int* lim() const { return reinterpret_cast<int*>(cols() + 8 * NT); }
  __device__ int* tok() const { return reinterpret_cast<int*>(cols() + 9 * NT); }
  __device__ float* nref() const { return cols() + 10 * NT; }  // minus ref()
};

// bf16: query rows of an entry into shared memory as the B operand of the score GEMM (K-major, 128-byte swizzle). Eight
// threads copy a row, 16 bytes at a time: chunk ch of a 128-byte block goes to chunk ch ^ (row % 8).
template <int NT>
__device__ __forceinline__ void load_query(const LatAttnParams& p, uint8_t* sq, const LatEntry& x, int t, int threads) {
  const int ch = t & 7;
  int tok = p.by_h(x.r0 + (t >> 3)), h = x.r0 + (t >> 3) - tok * p.H;
  const __nv_bfloat16* q = p.q + x.b * p.qs[0] + ch * 8;
#pragma unroll 1
  for (int row = t >> 3; row < NT; row += threads >> 3) {
    const bool there = x.r0 + row < p.R;
    const __nv_bfloat16* src = there ? q + tok * p.qs[1] + h * p.qs[2] : p.q;
    h += threads >> 3;
    while (h >= p.H) { h -= p.H; ++tok; }
    const uint32_t dst = smem_u32(sq) + row * 128 + (((ch ^ row) & 7) << 4);
#pragma unroll
    for (int i = 0; i < 9; ++i) cp_async16(dst + i * (NT * 128), src + (there ? i * 64 : 0), there ? 16u : 0u);
  }
  cp_async_wait_all();
}

// 8-bit: the split query. Rows come as they are by asynchronous copies, all of them in flight at once, each into the 1024 bytes
// that its two parts will take; then a warp converts row by row in place, 16 elements a lane (chunks lane and lane + 32 of 8).
// A row takes a warp 780 cycles, most of them in the conversions' pipe of its scheduler (32 rows by one warp: 25 000 cycles,
// more than everything else at the end of a piece), so rows are dealt to warps of all schedulers. A rolled loop keeps the code
// small: it is cold whenever it runs (16 rows unrolled: 20 000 cycles).
// Part i (0 .. 7) of 128 bytes of row `row`: high parts of blocks 0 .. 3, then low parts.
template <int NT>
__device__ __forceinline__ uint8_t* split_part(uint8_t* sq, int row, int i) {
  return sq + (i & 3) * (2 * NT * 128) + ((i >> 2) * NT + row) * 128;
}
template <int NT>
__device__ __forceinline__ void fetch_query_rows(const LatAttnParams& p, uint8_t* sq, const LatEntry& x, int row0, int end,
                                                 int step, int lane) {
  static_assert(NT <= 32, "a lane per row");
  // Lane = row: where each begins. Computed row by row in the loop, 32 of them took 15 000 cycles.
  const int tok = p.by_h(x.r0 + lane);
  const int64_t begins = tok * p.qs[1] + (x.r0 + lane - tok * p.H) * p.qs[2];
  const __nv_bfloat16* q = p.q + x.b * p.qs[0] + lane * 8;
#pragma unroll 1
  for (int row = row0; row < end; row += step) {
    const int64_t at = __shfl_sync(0xFFFFFFFFu, begins, row);
    const bool there = x.r0 + row < p.R;
    const __nv_bfloat16* src = there ? q + at : p.q;
    const uint32_t n = there ? 16u : 0u;
    cp_async16(smem_u32(split_part<NT>(sq, row, lane >> 3)) + (lane & 7) * 16, src, n);
    cp_async16(smem_u32(split_part<NT>(sq, row, 4 + (lane >> 3))) + (lane & 7) * 16, src + (there ? 256 : 0), n);
    if (lane < 8) cp_async16(smem_u32(sq) + NT * 1024 + row * 128 + (((lane ^ row) & 7) << 4), src + (there ? 512 : 0), n);
  }
  cp_async_wait_all();
}
template <int NT>
__device__ __forceinline__ void split_query_rows(uint8_t* sq, float* qk, int row0, int end, int step, int lane) {
#pragma unroll 2
  for (int row = row0; row < end; row += step) {
    const uint4 a = *reinterpret_cast<const uint4*>(split_part<NT>(sq, row, lane >> 3) + (lane & 7) * 16);
    const uint4 b = *reinterpret_cast<const uint4*>(split_part<NT>(sq, row, 4 + (lane >> 3)) + (lane & 7) * 16);
    __syncwarp();
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      top = fmax3(top, fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xFFFF0000u)));
    // magnitudes of floats order like their bits
    const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top));
    // the power of two that brings the row's largest element into (224, 448]
    int k = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7FFFFFu) > 0x600000u ? 7 : 8);
    k = bits == 0u ? 0 : max(k, -126);  // at most 120
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
    // an infinite element makes the row's scores NaN
    if (lane == 0) qk[row] = __uint_as_float(bits >= 0x7F800000u ? 0x7FC00000u : static_cast<uint32_t>(127 + k) << 23);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint16_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        split_e4m3x2(__uint_as_float(w[4 * i + j] << 16) * inv, __uint_as_float(w[4 * i + j] & 0xFFFF0000u) * inv, h[j], l[j]);
      const int ch = i * 32 + lane;  // elements [8 ch, 8 ch + 8): byte 8 (ch % 16) of block ch / 16
      const int at = (((((ch & 15) >> 1) ^ row) & 7) << 4) + (ch & 1) * 8;
      *reinterpret_cast<uint2*>(split_part<NT>(sq, row, ch >> 4) + at) =
          make_uint2(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16));
      *reinterpret_cast<uint2*>(split_part<NT>(sq, row, 4 + (ch >> 4)) + at) =
          make_uint2(l[0] | (static_cast<uint32_t>(l[1]) << 16), l[2] | (static_cast<uint32_t>(l[3]) << 16));
    }
  }
}

// Whether 16 bytes of the latent plane hold a value that is not finite: an e4m3 byte 0x7F or 0xFF, a bf16 exponent of ones.
// Adding one to it carries into the sign bit, which is masked out before.
template <bool FP8>
__device__ __forceinline__ bool not_finite(uint4 v) {
  constexpr uint32_t kMask = FP8 ? 0x7F7F7F7Fu : 0x7F807F80u, kOne = FP8 ? 0x01010101u : 0x00800080u;
  const uint32_t carry = ((v.x & kMask) + kOne) | ((v.y & kMask) + kOne) | ((v.z & kMask) + kOne) | ((v.w & kMask) + kOne);
  return (carry & ~kMask & (FP8 ? 0x80808080u : 0x80008000u)) != 0u;
}

// Softmax and epilogue of warpgroup g: columns [g CW, g CW + CW) of the row tile, thread = key of the tile (then output
// dimension) = TMEM lane.
template <int NT, bool FP8>
__device__ __forceinline__ void lat_softmax(const LatAttnParams& p, const LatShared<NT, FP8>& sm, const AbortCtl& ctl,
                                            LatWalk<NT> walk, uint32_t tmem, int g, int t) {
  using L = LatCfg<NT, FP8>;
  constexpr int NC = L::NC, CW = L::CW;
  constexpr int kStep = FP8 ? 32 : 16;      // keys of one MMA of the output GEMM
  constexpr float kRise = FP8 ? 4.f : 8.f;  // how far (log2) a score may exceed the reference
  constexpr int kOwn = CW > 32 ? CW / 32 : 1;
  const int w = t >> 5, lane = t & 31, cb = g * CW;
  const uint32_t bar = 1 + g;               // named barrier of this warpgroup; 3 = all softmax warpgroups
  const uint32_t tl = tmem + (static_cast<uint32_t>(w << 5) << 16);
  uint32_t tile = 0, slot0 = 0, piece = 0, loads = 0;  // loads: pieces with keys, whose queries are loaded
  int4 info = make_int4(-1, -1, -1, 0);
  while (walk.next(p)) {
    const LatEntry x = walk.x;
    const int tiles = walk.tiles();
    const bool whole = walk.begins && walk.ends;
    const int slot = 2 * blockIdx.x + (piece > 0 ? 1 : 0);
    if (!walk.begins) info.x = x.b * p.RT + x.r0 / NT;
    if (walk.begins && !walk.ends) { info.y = x.b * p.RT + x.r0 / NT; info.z = slot; }
    named_bar_sync(3, 128 * L::G);  // everybody has finished with the previous piece's columns
    const int prefix = max(x.len - x.nq, 0);
    if (g == 0 && t < 4) sm.poisoned()[t] = 0u;
    if (t < CW) {
      const int c = cb + t, r = x.r0 + c, tok = p.by_h(r);
      sm.tok()[c] = tok;
      // keys below the limit are visible; rows without a query are stored as zeros or not at all, whatever they see
      sm.lim()[c] = r >= p.R || tok >= x.nq ? 0x7FFFFFFF : p.tree != nullptr ? prefix : max(x.len - x.nq + tok + 1, 0);
      sm.ref()[c] = kNoRef;
      sm.nref()[c] = -kNoRef;
    }
    named_bar_sync(3, 128 * L::G);
    int min_lim = 0x7FFFFFFF;
#pragma unroll 8
    for (int c = 0; c < NT; ++c) min_lim = min(min_lim, sm.lim()[c]);
    if constexpr (L::kHelp) {
      if (tiles > 0) {  // the last score GEMM of the previous piece has completed: this warpgroup has read its scores
        uint8_t* sq = sm.base + L::kQOff;
        const int row0 = loader_rows(loads) + 4 * g + w;
        if (loads == 0) {
          fetch_query_rows<NT>(p, sq, x, row0, NT, 4 * L::G, lane);
          __syncwarp();
        } else {
          named_bar_sync(4, 128 * L::G + 32);
        }
        split_query_rows<NT>(sq, sm.qk(loads & 1), row0, NT, 4 * L::G, lane);
        fence_proxy_async_smem();
        mbar_arrive(sm.q_full());
      }
    }
    const float* qk = sm.qk(loads & 1) + cb;
    ++piece;
    if (tiles > 0) ++loads;
    float l[CW];
#pragma unroll
    for (int c = 0; c < CW; ++c) l[c] = 0.f;
    // score (log2) minus reference of four columns, two to an instruction
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    const auto above = [&](const float* sc, int c, float lk, float* d) {
      const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(sm.nref() + cb + c);
      uint64_t r0 = r.x, r1 = r.y;
      if (FP8) {
        const uint64_t lk2 = f2_pack(lk, lk);
        r0 = f2_add(r0, lk2);
        r1 = f2_add(r1, lk2);
      }
      f2_unpack(f2_fma(f2_pack(sc[c], sc[c + 1]), scale2, r0), d[0], d[1]);
      f2_unpack(f2_fma(f2_pack(sc[c + 2], sc[c + 3]), scale2, r1), d[2], d[3]);
    };

    // 8-bit: the factor of this thread's key is read a tile ahead, its page two tiles ahead.
    LatPage at(p, walk.k0 + t);
    int next_page = -1;
    float next_ks = 1.f;
    const auto fetch_page = [&](int n) { next_page = n < walk.k1 ? __ldg(p.table + x.b * p.table_stride + at.index) : -1; };
    const auto fetch_factor = [&](int n) {
      const bool there = next_page >= 0 && next_page < p.pages;
      next_ks = there ? p.scale[next_page * p.scale_stride[0] + at.row * p.scale_stride[1]] : 1.f;
      at.next_tile(p);
      fetch_page(n + kTile);
    };
    if (FP8) {
      fetch_page(walk.k0 + t);
      fetch_factor(walk.k0 + t);
    }
    for (int j = 0; j < tiles; ++j, ++tile) {
      const int n0 = walk.k0 + j * kTile, n = n0 + t;
      const uint32_t buf = tile % L::kScores;
      float ks = 1.f, lk = 0.f, iks = 1.f;  // the key's factor, its log2, its reciprocal
      // Half a step of 16 times a weight, 2^-14, times a number in [-1, 1) that is spread evenly over any run of keys: the weight
      // of a hidden key, 0, stays 0.
      const float offset = static_cast<float>(static_cast<int>(static_cast<uint32_t>(n) * 0x9E3779B9u)) * 0x1p-45f;
      bool bad_factor = false;  // not finite, or negative: the rows that see the key become NaN, and no others
      if (FP8) {
        if (n < walk.k1) {
          bad_factor = !(next_ks >= 0.f && next_ks < INFINITY);
          ks = bad_factor ? 1.f : fmaxf(next_ks, 0x1p-100f);  // the least that a write stores; the row sum holds its reciprocal
          lk = fast_log2(ks);
          iks = 1.f / ks;
        }
        fetch_factor(n + kTile);
      }
      const int end = min(walk.k1, n0 + kTile);
      // A tree's mask for this thread's key, a bit per column; its loads are all in flight at once, before the wait.
      uint32_t shown_to = 0xFFFFFFFFu;
      if (p.tree != nullptr && __any_sync(0xFFFFFFFFu, n >= min_lim && n < end)) {
        const bool in_tree = n >= min_lim && n < end;
        const uint8_t* mask = in_tree ? p.tree + x.b * p.tree_stride[0] + (n - (x.len - x.nq)) : p.tree;
        uint8_t m[CW];
#pragma unroll
        for (int c = 0; c < CW; ++c)
          m[c] = __ldg(mask + (in_tree && n >= sm.lim()[cb + c] ? sm.tok()[cb + c] * p.tree_stride[1] : 0));
        shown_to = 0u;
#pragma unroll
        for (int c = 0; c < CW; ++c) shown_to |= (n < sm.lim()[cb + c] || m[c] != 0 ? 1u : 0u) << c;
      }
      mbar_wait(sm.s_full(buf), (tile / L::kScores) & 1, ctl, 0x700);
      tc_fence_after_sync();
      float s[CW];  // scores before the softmax scale
      if (FP8) {
        uint32_t a[CW], b[CW], rp[CW];
        tmem_ld_cols<CW>(tl + kColS + buf * NC + cb, a);
        tmem_ld_cols<CW>(tl + kColS + buf * NC + NT + cb, b);
        tmem_ld_cols<CW>(tl + kColR + buf * NT + cb, rp);
        float f[CW];
#pragma unroll
        for (int c = 0; c < CW; c += 4) {
          const float4 q4 = *reinterpret_cast<const float4*>(qk + c);
          f[c] = q4.x * ks; f[c + 1] = q4.y * ks; f[c + 2] = q4.z * ks; f[c + 3] = q4.w * ks;
        }
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < CW; ++c)
          s[c] = fmaf(fmaf(__uint_as_float(b[c]), 0.0625f, __uint_as_float(a[c])), f[c], __uint_as_float(rp[c]));
      } else {
        uint32_t a[CW];
        tmem_ld_cols<CW>(tl + kColS + buf * NC + cb, a);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < CW; ++c) s[c] = __uint_as_float(a[c]);
      }
      if (FP8 && bad_factor) {
#pragma unroll
        for (int c = 0; c < CW; ++c) s[c] = __uint_as_float(0x7FC00000u);
      }
      if (n0 + kTile > min(min_lim, walk.k1)) {
        // Masked tile. The output GEMM takes the keys in steps of 16 (8-bit: 32); the rows of its last step that hold no
        // key of this piece are zeroed (0 * NaN would reach every output). A key that is hidden from some rows and not
        // finite is taken out of the tile and makes the rows that see it NaN.
        const int rows = (kStep - (end - n0) % kStep) % kStep;
#pragma unroll 1
        for (int i = g * 128 + t; i < rows * (FP8 ? 32 : 64); i += 128 * L::G) {
          const int row = end - n0 + i / (FP8 ? 32 : 64), ch = i % (FP8 ? 32 : 64);
          *reinterpret_cast<uint4*>(sm.base + ((slot0 + ch / (FP8 ? 8 : 16)) % L::NS) * L::kSlot +
                                    (FP8 ? 0 : (ch >> 3 & 1) * 16384) + row * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        bool poison = false;
        if (end > min_lim) {
          constexpr int kChunks = FP8 ? 32 : 64;  // of 16 bytes in a key's latent vector
          const auto chunk = [&](int row, int ch) {
            return reinterpret_cast<uint4*>(sm.base + ((slot0 + ch / (kChunks / 4)) % L::NS) * L::kSlot +
                                            (FP8 ? 0 : (ch >> 3 & 1) * 16384) + row * 128 + (ch & 7) * 16);
          };
          const int row0 = max(min_lim - n0, 0);
#pragma unroll 1
          for (int i = g * 128 + t; i < (end - n0 - row0) * kChunks; i += 128 * L::G) {
            const int row = row0 + i / kChunks;
            if (not_finite<FP8>(*chunk(row, i % kChunks))) atomicOr(sm.poisoned() + (row >> 5), 1u << (row & 31));
          }
          named_bar_sync(3, 128 * L::G);
          const uint4 found = *reinterpret_cast<const uint4*>(sm.poisoned());
          if (L::G > 1) named_bar_sync(3, 128 * L::G);  // both warpgroups have read it before either sets a bit of the next tile
          if ((found.x | found.y | found.z | found.w) != 0u) {
            poison = (sm.poisoned()[w] >> lane & 1u) != 0u;
            named_bar_sync(3, 128 * L::G);
            if (g == 0 && t < 4) sm.poisoned()[t] = 0u;
            named_bar_sync(3, 128 * L::G);
            if (poison)
#pragma unroll 1
              for (int i = 0; i < kChunks; ++i) *chunk(t, i) = make_uint4(0, 0, 0, 0);
          }
        }
        const float shown = __uint_as_float(0x7FC00000u);
        if (p.tree == nullptr) {
#pragma unroll
          for (int c = 0; c < CW; ++c) s[c] = n < min(end, sm.lim()[cb + c]) ? (poison ? shown : s[c]) : -INFINITY;
        } else {
#pragma unroll
          for (int c = 0; c < CW; ++c) s[c] = n < end && (shown_to >> c & 1u) != 0u ? (poison ? shown : s[c]) : -INFINITY;
        }
        __syncwarp();
      }
      float rise = -INFINITY;
#pragma unroll
      for (int c = 0; c < CW; c += 4) {
        float d[4];
        above(s, c, lk, d);
        rise = fmax3(fmax3(rise, d[0], d[1]), d[2], d[3]);
      }
      if (named_bar_or(bar, 128, rise > kRise)) {
        {
          float m[CW];
#pragma unroll
          for (int c = 0; c < CW; ++c) m[c] = fmaf(s[c], p.scale_log2, lk);
          reduce_cols<CW, true>(m, lane);
#pragma unroll
          for (int i = 0; i < kOwn; ++i) sm.red(g)[w * CW + first_column<CW>(lane) + i] = m[i];
        }
        named_bar_sync(bar, 128);
        if (t < CW) {
          const float old = sm.ref()[cb + t];
          const float* red = sm.red(g) + t;
          const float m = fmaxf(fmaxf(fmaxf(red[0], red[CW]), fmaxf(red[2 * CW], red[3 * CW])), old);
          sm.ref()[cb + t] = m;
          sm.nref()[cb + t] = -m;
          sm.fac()[cb + t] = fast_exp2(old - m);
        }
        named_bar_sync(bar, 128);
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < CW; ++c) l[c] *= sm.fac()[cb + c];
          mbar_wait(sm.o_full(tile - 1), ((tile - 1) >> 1) & 1, ctl, 0x780);  // O^T of the tiles so far
          tc_fence_after_sync();
#pragma unroll 1
          for (int i = 0; i < 4 * NC; i += 16) {
            const int c0 = i % NT;  // hi and lo columns alike
            if (L::G > 1 && c0 / CW != g) continue;
            uint32_t o[16];
            tmem_ld16(tl + i, o);
            tmem_wait_ld();
            const float* f = sm.fac() + c0;
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f[c]);
            tmem_st16(tl + i, o);
          }
          tmem_wait_st();
        }
      }
      // 8-bit: this tile's buffer of weights was last read by the output GEMM two tiles ago. The score GEMM's commit does not
      // stand in for that one: without this wait, and with one barrier for the rescale's, sums were lost.
      if (FP8 && tile >= 2) mbar_wait(sm.o_full(tile), ((tile - 2) >> 1) & 1, ctl, 0x790);
      // P^T is the B operand of the output GEMM as it comes: a key's weights are contiguous (MN-major), rows of kPRow bytes
      // with the swizzle of that width.
      uint8_t* sp = sm.base + L::kPOff + (FP8 ? (tile & 1) * L::kP : 0) + t * L::kPRow;
      const int twist = L::kPRow == 128 ? t & 7 : L::kPRow == 64 ? (t >> 1) & 3 : (t >> 2) & 1;
#pragma unroll
      for (int c0 = 0; c0 < CW; c0 += 16) {
        float pw[16];
#pragma unroll
        for (int c = 0; c < 16; c += 4) above(s, c0 + c, lk, pw + c);
#pragma unroll
        for (int c = 0; c < 16; ++c) pw[c] = fast_exp2(pw[c]);
        if (FP8) {
          // 16 times the weight, at most 256; the remainder of its first rounding is at most 16, times 16
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            f2_unpack(f2_fma(f2_pack(pw[c], pw[c + 1]), f2_pack(iks, iks), f2_pack(l[c0 + c], l[c0 + c + 1])), l[c0 + c],
                      l[c0 + c + 1]);
            uint16_t h, r;
            split_e4m3x2(fmaf(pw[c], 16.f, offset), fmaf(pw[c + 1], 16.f, offset), h, r);
            hi[c >> 2] = (c & 2) ? hi[c >> 2] | (static_cast<uint32_t>(h) << 16) : h;
            lo[c >> 2] = (c & 2) ? lo[c >> 2] | (static_cast<uint32_t>(r) << 16) : r;
          }
          const int ch = (cb + c0) >> 4;
          *reinterpret_cast<uint4*>(sp + ((ch ^ twist) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(sp + (((ch + NT / 16) ^ twist) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        } else {
          uint32_t w2[8];
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            f2_unpack(f2_add(f2_pack(l[c0 + c], l[c0 + c + 1]), f2_pack(pw[c], pw[c + 1])), l[c0 + c], l[c0 + c + 1]);
            w2[c >> 1] = pack_bf16(pw[c], pw[c + 1]);
          }
          const int ch = (cb + c0) >> 3;
          *reinterpret_cast<uint4*>(sp + ((ch ^ twist) << 4)) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
          *reinterpret_cast<uint4*>(sp + (((ch + 1) ^ twist) << 4)) = make_uint4(w2[4], w2[5], w2[6], w2[7]);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      mbar_arrive(sm.p_full(tile));
      slot0 = (slot0 + 4) % L::NS;
    }

    // ---- epilogue: thread = output dimension
    reduce_cols<CW, false>(l, lane);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sm.red(g)[w * CW + first_column<CW>(lane) + i] = l[i];
    named_bar_sync(bar, 128);
    float sum = 0.f;
    if (t < CW) {
      const float* red = sm.red(g) + t;
      const bool query = sm.tok()[cb + t] < x.nq;
      sum = query ? (red[0] + red[CW]) + (red[2 * CW] + red[3 * CW]) : 0.f;
      if (!query) sm.ref()[cb + t] = kNoRef;
      sm.fac()[cb + t] = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
    }
    named_bar_sync(bar, 128);
    if (tiles > 0) {
      mbar_wait(sm.o_full(tile - 1), ((tile - 1) >> 1) & 1, ctl, 0x800);
      tc_fence_after_sync();
    }
    // Rolled loops: the code runs once per piece, and unrolled it waited for the instruction cache at every store.
    const int rows = min(p.R - x.r0, NT);
#pragma unroll 1
    for (int i = 0; i < 4 * CW; i += 32) {
      uint32_t o[32], lo[32];
      float y[32];
      if (tiles > 0) {
#pragma unroll
        for (int u = 0; u < 32; u += 16) {
          const uint32_t at = tl + (i + u) / CW * NC + cb + (i + u) % CW;
          tmem_ld16(at, o + u);
          if (FP8) tmem_ld16(at + NT, lo + u);
        }
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          y[c] = __uint_as_float(o[c]);
          if (FP8) y[c] = fmaf(__uint_as_float(lo[c]), 0.0625f, y[c]) * 0.0625f;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) y[c] = 0.f;
      }
      if (!whole) {
        // [column / 4][dimension][4 columns]: 16 bytes a lane, neighbouring. Rows without a query may hold anything.
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const int d0 = (i + c) / CW * 128 + t, c0 = cb + (i + c) % CW;
          *(reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(slot) * NT + c0) * kLat) + d0) =
              make_float4(y[c], y[c + 1], y[c + 2], y[c + 3]);
        }
        continue;
      }
#pragma unroll
      for (int u = 0; u < 32; u += 16) {
        const int d0 = (i + u) / CW * 128 + t, c0 = cb + (i + u) % CW;
#pragma unroll
        for (int c = u; c < u + 16; ++c) {
          const float f = sm.fac()[c0 + c - u];
          y[c] = f == 0.f ? 0.f : y[c] * f;  // no key, or no query (whose scores may be anything)
        }
        // neighbouring lanes trade: the even one stores two dimensions of an even column, the odd one of the next column
        const int odd = t & 1;
        __nv_bfloat16* d = p.out + (static_cast<int64_t>(x.b) * p.R + x.r0 + c0 + odd) * kLat + (d0 & ~1);
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? y[u + c] : y[u + c + 1], 1);
          const uint32_t pair = odd ? pack_bf16(got, y[u + c + 1]) : pack_bf16(y[u + c], got);
          if (c0 + c + odd < rows) *reinterpret_cast<uint32_t*>(d + c * kLat) = pair;
        }
      }
    }
    if (t < CW) {
      const int c = cb + t, r = x.r0 + c;
      if (!whole) {
        p.part_ml[slot * NT + c] = make_float2(sm.ref()[c], sum);
      } else if (p.lse != nullptr && r < p.R) {
        const int tok = p.by_h(r);
        p.lse[static_cast<int64_t>(x.b) * p.R + static_cast<int64_t>(r - tok * p.H) * p.Sq + tok] =
            sum == 0.f ? -INFINITY : sm.ref()[c] + log2f(sum);
      }
    }
    tc_fence_before_sync();
  }
  if (g == 0 && t == 0 && p.part_info != nullptr) p.part_info[blockIdx.x] = info;
}

template <int NT, bool FP8>
__global__ void __launch_bounds__(LatCfg<NT, FP8>::kThreads, 1)
    latent_attn_kernel(const __grid_constant__ CUtensorMap tm_lat, const __grid_constant__ CUtensorMap tm_rope,
                       const LatAttnParams p) {
  using L = LatCfg<NT, FP8>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const LatShared<NT, FP8> sm(smem);
  uint32_t* tmem_slot = sm.tmem_slot();
  volatile uint32_t* abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AbortCtl ctl{p.status, abort_flag};

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::NS; ++i) { mbar_init(sm.full(i), 1); mbar_init(sm.empty(i), 1); }
    mbar_init(sm.rfull(), 1);
    mbar_init(sm.rempty(), 1);
    mbar_init(sm.q_full(), 32 * L::kLoadWarps + (L::kHelp ? 128 * L::G : 0));
    mbar_init(sm.q_empty(), 1);
    mbar_init(sm.s_full(0), 1);
    mbar_init(sm.s_full(1), 1);
    mbar_init(sm.p_full(0), 128 * L::G);
    mbar_init(sm.p_full(1), 128 * L::G);
    mbar_init(sm.o_full(0), 1);
    mbar_init(sm.o_full(1), 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 96) {
    tma_prefetch_desc(&tm_lat);
    tma_prefetch_desc(&tm_rope);
  }
  if (threadIdx.x == 64)  // a launch that finds an error already recorded does no work
    *abort_flag = (p.status != nullptr && *reinterpret_cast<volatile uint32_t*>(p.status) != 0u) ? 1u : 0u;
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // the merge kernel may be set up; it waits for this grid's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int entries = p.B * p.RT, me = static_cast<int>(blockIdx.x);
  const auto check_lengths = [&](const LatEntry& x) {
    if (x.r0 != 0) return;
    const int len = __ldg(p.lens + x.b);
    if (len < 0 || len > p.max_keys || (p.qlens != nullptr && (__ldg(p.qlens + x.b) < 0 || __ldg(p.qlens + x.b) > p.Sq)))
      if (p.status != nullptr) atomicCAS(p.status, 0u, (kErrIndex << 24) | kIdxLength);
  };
  LatWalk<NT> walk;
  if (p.whole && entries == static_cast<int>(gridDim.x)) {  // each entry has a CTA of its own
    const LatEntry x = lat_entry<NT>(p, me);
    if (threadIdx.x == 0) check_lengths(x);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    walk.e = me;
    walk.off = 0;
    walk.left = 1;
    walk.extra = 0;
  } else {
    // This CTA's share of the work line: every thread counts a run of entries, then a scan over the CTA.
    const int run = (entries + L::kThreads - 1) / L::kThreads;
    const int e_begin = min(static_cast<int>(threadIdx.x) * run, entries), e_end = min(e_begin + run, entries);
    int mine = 0;
    for (int e = e_begin; e < e_end; ++e) {
      const LatEntry x = lat_entry<NT>(p, e);
      mine += lat_units(p, x.keys);
      if (blockIdx.x == 0) check_lengths(x);
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += v;
    }
    int* scan = sm.scan();
    if (lane == 31) scan[warp] = incl;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    int before = 0, units = 0;
#pragma unroll
    for (int i = 0; i < L::kThreads / 32; ++i) {
      if (i < warp) before += scan[i];
      units += scan[i];
    }
    // Every entry takes L::kExtra more places; not where every unit can have a CTA of its own.
    const int extra = units <= static_cast<int>(gridDim.x) ? 0 : L::kExtra;
    const int total = units + extra * entries;
    // with fewer places than CTAs the first ones get one each: the CTAs of an entry are always neighbours
    const int busy = min(total, static_cast<int>(gridDim.x));
    const int share = total / busy, more = total - share * busy;
    const int u0 = me < busy ? me * share + min(me, more) : total, u1 = me < busy ? u0 + share + (me < more ? 1 : 0) : total;
    {
      mine += extra * (e_end - e_begin);
      int at = before + incl + extra * e_end - mine;  // places in front of this thread's entries
      if (u0 < u1 && at <= u0 && u0 < at + mine) {
        int e = e_begin;
        while (true) {
          const int n = lat_units(p, lat_entry<NT>(p, e).keys) + extra;
          if (u0 < at + n) break;
          at += n;
          ++e;
        }
        scan[12] = e;
        scan[13] = u0 - at;
      }
    }
    __syncthreads();
    walk.e = u0 < u1 ? scan[12] : 0;
    walk.off = u0 < u1 ? scan[13] : 0;
    walk.left = u1 - u0;
    walk.extra = extra;
  }
  const uint32_t tmem = *tmem_slot;
  bool healthy = *abort_flag == 0u;
  if ((smem_u32(smem) & 1023u) != 0u) {  // the swizzled tiles need a 1024-byte aligned window
    if (threadIdx.x == 0) report_error(ctl, kErrSmemAlign, smem_u32(smem));
    healthy = false;
  }
  if (!healthy) walk.left = 0;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer: one lane per page of the tile
    const int box = min(p.page_size, kBox);
    uint32_t it = 0, tile = 0;
    while (walk.next(p)) {
      const int32_t* table = p.table + walk.x.b * p.table_stride;
      LatPage at(p, walk.k0 + lane * box);
      int next_page = 0;  // of the next tile, read a tile ahead
      if (lane * box < min(kTile, walk.k1 - walk.k0)) next_page = __ldg(table + at.index);
      for (int j = 0; j < walk.tiles(); ++j, ++tile) {
        const int n0 = walk.k0 + j * kTile;
        const int boxes = (min(kTile, walk.k1 - n0) + box - 1) / box;
        const int row = at.row;
        int page = next_page;
        at.next_tile(p);
        if (lane * box < min(kTile, walk.k1 - n0 - kTile)) next_page = __ldg(table + at.index);
        if (lane < boxes) {
          if (page < 0 || page >= p.pages) {
            if (p.status != nullptr) atomicCAS(p.status, 0u, (kErrIndex << 24) | kIdxPage);
            page = 0;
          }
        }
        for (int i = 0; i < 4; ++i, ++it) {
          const uint32_t s = it % L::NS;
          mbar_wait(sm.empty(s), ((it / L::NS) & 1) ^ 1, ctl, 0x100 + s);
          if (lane == 0) mbar_arrive_expect_tx(sm.full(s), boxes * box * (FP8 ? 128 : 256));
          __syncwarp();
          if (lane < boxes) {
            uint8_t* dst = smem + s * L::kSlot + lane * box * 128;
            tma_load_4d(dst, &tm_lat, sm.full(s), i * 128, 0, row, page);
            if (!FP8) tma_load_4d(dst + 16384, &tm_lat, sm.full(s), i * 128 + 64, 0, row, page);
          }
        }
        // The rope tile comes last, as its place is free last: once the previous tile's score GEMM (8-bit) or output GEMM (whose
        // weights lie there) has completed.
        mbar_wait(sm.rempty(), (tile & 1) ^ 1, ctl, 0x200);
        if (lane == 0) mbar_arrive_expect_tx(sm.rfull(), boxes * box * 128);
        __syncwarp();
        if (lane < boxes) tma_load_4d(smem + L::kRopeOff + lane * box * 128, &tm_rope, sm.rfull(), 0, 0, row, page);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ score GEMM, one thread
    // An MMA of these sizes takes 40 to 65 cycles, no longer than a warp needs to form its descriptors and agree on a lane, so
    // one thread of a warp does all, and the two GEMMs, which wait for different things, are issued by two warps. With one
    // warp for both, the tensor pipe waited half of the time for the next instruction. The steps are rolled loops where they
    // wait: their code runs once a tile between that of the softmax warps, and every jump over an unrolled copy waited for
    // the instruction cache.
    if (elect_one()) {
      constexpr uint32_t id_rope = make_idesc_bf16(128, NT, false, false);
      constexpr uint32_t id_qk = FP8 ? make_idesc_e4m3(128, L::NC, false) : id_rope;
      const uint64_t q_desc = make_smem_desc(smem_u32(smem + L::kQOff), 16, 1024);
      const uint64_t qr_desc = make_smem_desc(smem_u32(smem + L::kQOff + L::kQLat), 16, 1024);
      const uint64_t k_desc = make_smem_desc(smem_u32(smem), 16, 1024);  // K-major: keys x dims
      const uint64_t r_desc = make_smem_desc(smem_u32(smem + L::kRopeOff), 16, 1024);
      uint32_t ks = 0, kph = 0, tile = 0, q_phase = 0;
      while (walk.next(p)) {
        const int tiles = walk.tiles();
        if (tiles > 0) {
          mbar_wait(sm.q_full(), q_phase, ctl, 0x300);
          q_phase ^= 1;
        }
        for (int j = 0; j < tiles; ++j, ++tile) {
          // The weights of the tile that used this buffer of S^T last are written, so its scores have been read; at a piece's
          // first tile, those of the previous piece's last one (its query factors may then be replaced).
          const uint32_t before = j == 0 ? 1 : L::kScores;
          if (tile >= before) mbar_wait(sm.p_full(tile - before), ((tile - before) >> 1) & 1, ctl, 0x680);
          const uint32_t buf = tile % L::kScores;
          const uint32_t d = tmem + kColS + buf * L::NC;
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {  // 128 latent dimensions each
            mbar_wait(sm.full(ks), kph, ctl, 0x400 + ks);
            tc_fence_after_sync();
            const uint64_t kd = desc_at(k_desc, ks * L::kSlot), qd = desc_at(q_desc, i * (2 * NT * 128));
            if (FP8) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_ss_f8(d, desc_at(kd, k * 32), desc_at(qd, k * 32), id_qk, (i > 0 || k > 0) ? 1u : 0u);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                umma_ss(d, desc_at(kd, (k >> 2) * 16384 + (k & 3) * 32), desc_at(qd, (k >> 2) * (NT * 128) + (k & 3) * 32),
                        id_qk, (i > 0 || k > 0) ? 1u : 0u);
            }
            if (++ks == L::NS) { ks = 0; kph ^= 1; }
          }
          mbar_wait(sm.rfull(), tile & 1, ctl, 0x500);
          tc_fence_after_sync();
          const uint32_t dr = FP8 ? tmem + kColR + buf * NT : d;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_ss(dr, desc_at(r_desc, k * 32), desc_at(qr_desc, k * 32), id_rope, (!FP8 || k > 0) ? 1u : 0u);
          umma_commit(sm.s_full(buf));
          if (FP8) umma_commit(sm.rempty());
          if (j + 1 == tiles) umma_commit(sm.q_empty());
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ output GEMM, one thread
    if (elect_one()) {
      constexpr uint32_t id_pv = FP8 ? make_idesc_e4m3(128, L::NC, true) : make_idesc_bf16(128, NT, true, true);
      const uint64_t p_desc = make_row_desc(smem_u32(smem + L::kPOff), L::kPRow);
      const uint64_t v_desc = make_smem_desc(smem_u32(smem), 16384, 1024);  // MN-major: dims x keys
      uint32_t vs = 0, tile = 0;
      while (walk.next(p)) {
        const int tiles = walk.tiles(), keys = walk.k1 - walk.k0;
        for (int j = 0; j < tiles; ++j, ++tile) {
          const uint64_t pd = FP8 ? desc_at(p_desc, (tile & 1) * L::kP) : p_desc;
          const int steps = (min(keys - j * kTile, kTile) + (FP8 ? 31 : 15)) / (FP8 ? 32 : 16);
          mbar_wait(sm.p_full(tile), (tile >> 1) & 1, ctl, 0x600);
          tc_fence_after_sync();
          const auto output_gemm = [&](auto all) {
            constexpr int kSteps = FP8 ? 4 : 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t slot = L::NS == 4 ? i : vs;
              if (++vs == L::NS) vs = 0;
              const uint64_t vd = desc_at(v_desc, slot * L::kSlot);
#pragma unroll(decltype(all)::value ? kSteps : 1)
              for (int k = 0; k < (decltype(all)::value ? kSteps : steps); ++k) {
                if (FP8)
                  umma_ss_f8(tmem + i * L::NC, desc_at(vd, k * 4096), desc_at(pd, k * 32 * L::kPRow), id_pv,
                             (j > 0 || k > 0) ? 1u : 0u);
                else
                  umma_ss(tmem + i * L::NC, desc_at(vd, k * 2048), desc_at(pd, k * 16 * L::kPRow), id_pv,
                          (j > 0 || k > 0) ? 1u : 0u);
              }
              umma_commit(sm.empty(slot));
            }
          };
          if (steps == (FP8 ? 4 : 8)) output_gemm(Int<1>());
          else output_gemm(Int<0>());  // the last tile of a piece may need fewer steps of keys
          if (!FP8) umma_commit(sm.rempty());
          umma_commit(sm.o_full(tile));
        }
      }
    }
  } else if (warp >= 4 && warp < 4 + 4 * L::G) {
    lat_softmax<NT, FP8>(p, sm, ctl, walk, tmem, (warp - 4) >> 2, static_cast<int>(threadIdx.x) & 127);
  } else {
    // ------------------------------------------------------------------ query loaders, one piece ahead
    const int loader = warp < 4 ? 0 : warp - 3 - 4 * L::G;
    // Query factors alternate between two places by the pieces that have keys: one without may lie between two that do, and
    // the softmax may still be reading those of the piece before it.
    uint32_t q_phase = 1, loads = 0;
    while (walk.next(p)) {
      const int tiles = walk.tiles();
      if (tiles > 0) {
        uint8_t* sq = smem + L::kQOff;
        mbar_wait(sm.q_empty(), q_phase, ctl, 0x380);  // the previous piece's last score GEMM has read its query
        if constexpr (L::kHelp) {  // the softmax warps fetch their own rows of a CTA's first query, and find those of later ones
          fetch_query_rows<NT>(p, sq, walk.x, 0, loads == 0 ? loader_rows(0) : NT, 1, lane);
          if (loads > 0) asm volatile("bar.arrive 4, %0;" ::"n"(128 * L::G + 32) : "memory");
          __syncwarp();
          split_query_rows<NT>(sq, sm.qk(loads & 1), 0, loader_rows(loads), 1, lane);
        } else if constexpr (FP8) {
          fetch_query_rows<NT>(p, sq, walk.x, loader, NT, L::kLoadWarps, lane);
          __syncwarp();
          split_query_rows<NT>(sq, sm.qk(loads & 1), loader, NT, L::kLoadWarps, lane);
        } else {
          load_query<NT>(p, sq, walk.x, loader * 32 + lane, L::kLoadWarps * 32);
        }
        q_phase ^= 1;
        fence_proxy_async_smem();
        mbar_arrive(sm.q_full());
        ++loads;
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {  // let copies and MMAs still in flight drain before shared memory and TMEM are handed back
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Merge of a row tile that several CTAs worked on: out = sum_i 2^(ref_i - M) O_i / sum_i 2^(ref_i - M) l_i, in key order.
// Block (j, four columns): the j-th entry that a CTA began and did not finish; there are at most as many as entries, and
// one less than CTAs. A thread has one output dimension of the four columns, and the parts are dealt to SPLIT groups of
// threads: 1 for many entries, which have few parts each, 4, or 16 for a long context cut into many parts (100 000 keys of one
// sequence, 148 parts: 42 us with 4, 37 with 16; 16 sequences x 64 rows, 9 parts: 47 us with 1, 49.5 with 4, 68 with 16). The
// launch is a programmatic one: it waits for the attention kernel's results in the kernel instead of before it.
constexpr int kMergeThreads = 512;
template <int NT, int SPLIT>
__global__ void __launch_bounds__(kMergeThreads) latent_merge_kernel(const LatAttnParams p, int ctas) {
  __shared__ int warp_jobs[16];
  __shared__ int job[2];  // CTA, slot
  __shared__ int entry;
  __shared__ uint32_t failed;  // read once: another stream may record an error between two threads' reads of the word
  __shared__ float4 wt[kMergeThreads];
  __shared__ float4 red[2][1];
  constexpr int kGroup = kMergeThreads / SPLIT;
  __shared__ float4 acc_s[SPLIT > 1 ? kMergeThreads : 1];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int c4 = blockIdx.y;  // columns [4 c4, 4 c4 + 4)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (t == 0) failed = p.status != nullptr ? *reinterpret_cast<volatile uint32_t*>(p.status) : 0u;
  const int4 info = t < ctas ? p.part_info[t] : make_int4(-1, -1, -1, 0);
  const uint32_t begun = __ballot_sync(0xFFFFFFFFu, info.y >= 0);
  if (lane == 0) warp_jobs[warp] = __popc(begun);
  __syncthreads();
  int rank = __popc(begun & ((1u << lane) - 1u)), jobs = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (i < warp) rank += warp_jobs[i];
    jobs += warp_jobs[i];
  }
  if (failed != 0u || static_cast<int>(blockIdx.x) >= jobs) return;
  if (info.y >= 0 && rank == static_cast<int>(blockIdx.x)) { job[0] = t; job[1] = info.z; entry = info.y; }
  __syncthreads();
  const int c = job[0], e = entry;
  // parts: the slot of CTA c, then the first slot of each following CTA that continues the entry
  const int n = 1 + __syncthreads_count(t > c && info.x == e);
  const auto slot_of = [&](int i) { return i == 0 ? job[1] : 2 * (c + i); };
  // Weights of the parts, by the first 128 threads: lane group of 32 = column, each column's parts over its lanes.
  if (warp < 4) {
    const float2* ml = p.part_ml + 4 * c4 + warp;
    float top = kNoRef;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, ml[slot_of(i) * NT].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    float sum = 0.f;
    for (int i = lane; i < n; i += 32) {
      const float2 v = ml[slot_of(i) * NT];
      const float w = fast_exp2(v.x - top);
      reinterpret_cast<float*>(wt + i)[warp] = w;
      sum += w * v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) {
      reinterpret_cast<float*>(&red[0][0])[warp] = sum;
      reinterpret_cast<float*>(&red[1][0])[warp] = top;
    }
  }
  __syncthreads();
  const int g = t / kGroup, d = blockIdx.z * kGroup + t % kGroup;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = g; i < n; i += SPLIT) {
    const float4 f = wt[i];
    const float4 v = *(reinterpret_cast<const float4*>(p.part_o + (static_cast<int64_t>(slot_of(i)) * NT + 4 * c4) * kLat) + d);
    acc.x = fmaf(f.x, v.x, acc.x); acc.y = fmaf(f.y, v.y, acc.y); acc.z = fmaf(f.z, v.z, acc.z); acc.w = fmaf(f.w, v.w, acc.w);
  }
  if (SPLIT > 1) {
    acc_s[t] = acc;
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int i = 1; i < SPLIT; ++i) {
      const float4 v = acc_s[i * kGroup + t];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
  }
  // (plain divisions here: with FastDiv's the merge of one sequence's 148 parts took 14.7 instead of 12.1 us)
  const int b = e / p.RT, r0 = (e - b * p.RT) * NT + 4 * c4;
  const float sums[4] = {red[0][0].x, red[0][0].y, red[0][0].z, red[0][0].w};
  const float sum_top[4] = {red[1][0].x, red[1][0].y, red[1][0].z, red[1][0].w};
  const float o[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + i;
    if (r >= p.R) break;
    const bool none = sums[i] == 0.f;  // no key, or no query
    p.out[(static_cast<int64_t>(b) * p.R + r) * kLat + d] = __float2bfloat16_rn(none ? 0.f : o[i] / sums[i]);
    if (d == 0 && p.lse != nullptr) {
      const int tok = r / p.H;
      p.lse[static_cast<int64_t>(b) * p.R + static_cast<int64_t>(r - tok * p.H) * p.Sq + tok] =
          none ? -INFINITY : sum_top[i] + log2f(sums[i]);
    }
  }
}

// Rows per tile: the least that holds a sequence's rows. 64 (8-bit: 32, its columns count twice) is what TMEM and shared
// memory hold beside a whole 128-key tile.
static int lat_rows(int64_t rows, bool fp8) { return rows <= 16 ? 16 : rows <= 32 || fp8 ? 32 : 64; }

// Keys per unit of work, and CTAs. The unit is 64 keys. Where no sequence can pass one tile, and where cutting would not pay
// for the merge, it is all of a sequence: nothing is cut then, and one launch does. With a CTA for each of E entries of at
// most T tiles, cutting saves up to T (1 - E / SMs) tiles; the merge takes about as long as 3.6 tiles in bf16 and 6.6 in 8
// bits (and another launch from the host). Measured, cut against whole, 16 heads, us: bf16, one sequence of 256 keys 10.2 and
// 9.3, of 512 keys 10.9 and 13, 148 of up to 512 26.9 and 20.0, of up to 1024 36.1 and 31.5; 8-bit, one of 512 keys 11.3 and
// 11.2, of 1024 11.8 and 15, 148 of up to 1024 26.8 and 20.1. The lengths behind E are not known here, so sequences
// of more than 1024 keys are always cut.
constexpr int kWhole = 1024;
struct LatPlan { int unit_log2, ctas; };
static int lat_plan(int64_t entries, int64_t max_keys, bool fp8, LatPlan* plan) {
  int dev = 0, sms = 148;
  PITH_CUDA(cudaGetDevice(&dev));
  PITH_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  if (sms > kMergeThreads) sms = kMergeThreads;  // the merge looks at one CTA per thread
  const int64_t tiles = (max_keys + kTile - 1) / kTile;
  const bool whole = max_keys <= kWhole && entries <= sms && tiles * (sms - entries) * 10 <= sms * (fp8 ? 66 : 36);
  plan->unit_log2 = max_keys <= kTile ? 7 : whole ? 10 : 6;
  const int64_t unit = 1ll << plan->unit_log2, units = entries * (max_keys <= unit ? 1 : (max_keys + unit - 1) / unit);
  plan->ctas = static_cast<int>(units < sms ? units : sms);
  return kOk;
}

template <int NT, bool FP8>
static int launch_latent_attn(const pith_latent_attn_args* a, LatAttnParams& p, int ctas, cudaStream_t st) {
  using L = LatCfg<NT, FP8>;
  CUtensorMap tl, tr;
  const pith_latent_cache& c = a->cache;
  const int64_t ls[3] = {axis_stride(c.pages, c.latent_stride[0], c.page_size * c.latent_stride[1]), c.latent_stride[1], kLat};
  const int64_t rs[3] = {axis_stride(c.pages, c.rope_stride[0], c.page_size * c.rope_stride[1]), c.rope_stride[1], kRp};
  const int box = c.page_size < kBox ? c.page_size : kBox;
  if (int rc = make_tensor_map(&tl, c.latent, FP8 ? 1 : 2, c.pages, c.page_size, 1, kLat, ls, FP8 ? 128 : 64, box)) return rc;
  if (int rc = make_tensor_map(&tr, c.rope, 2, c.pages, c.page_size, 1, kRp, rs, 64, box)) return rc;
  auto kern = latent_attn_kernel<NT, FP8>;
  PITH_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc));
  kern<<<ctas, L::kThreads, L::kAlloc, st>>>(tl, tr, p);
  PITH_CUDA(cudaGetLastError());
  if (!p.whole) {  // an entry of one unit is never cut
    const int64_t entries = static_cast<int64_t>(p.B) * p.RT;
    cudaLaunchConfig_t cfg = {};
    const unsigned jobs = static_cast<unsigned>(entries < ctas - 1 ? entries : ctas - 1);
    const unsigned cols = static_cast<unsigned>((p.R < NT ? p.R : NT) + 3) / 4;
    const int split = entries * 10 >= ctas ? 1 : entries * 32 >= ctas ? 4 : 16;  // by the parts of an entry
    cfg.gridDim = dim3(jobs, cols, split);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    auto merge = split == 1 ? latent_merge_kernel<NT, 1> : split == 4 ? latent_merge_kernel<NT, 4> : latent_merge_kernel<NT, 16>;
    PITH_CUDA(cudaLaunchKernelEx(&cfg, merge, static_cast<const LatAttnParams&>(p), ctas));
  }
  return kOk;
}

}  // namespace pith

using namespace pith;

extern "C" size_t pith_latent_attn_workspace_bytes(int32_t B, int32_t Sq, int32_t H, int64_t max_keys, int32_t dtype) {
  if (B <= 0 || Sq <= 0 || H <= 0) return 0;
  const int nt = lat_rows(static_cast<int64_t>(Sq) * H, dtype == PITH_DTYPE_E4M3);
  LatPlan plan;
  if (lat_plan(static_cast<int64_t>(B) * ((static_cast<int64_t>(Sq) * H + nt - 1) / nt), max_keys,
               dtype == PITH_DTYPE_E4M3, &plan))
    return 0;
  if (max_keys <= (1ll << plan.unit_log2)) return 0;  // no entry is ever cut
  return static_cast<size_t>(plan.ctas) * (2 * nt * (kLat * 4 + 8) + 16);
}

extern "C" int pith_latent_attn(const pith_latent_attn_args* a, void* stream) {
  PITH_REQUIRE(a != nullptr, "null args");
  PITH_REQUIRE(a->B >= 0 && a->Sq >= 0 && a->H >= 0, "negative size");
  if (int rc = check_latent_cache(a->cache)) return rc;
  PITH_REQUIRE(a->softmax_scale > 0.f, "softmax_scale must be positive");
  if (a->B == 0 || a->Sq == 0 || a->H == 0) return kOk;
  PITH_REQUIRE(a->q && a->out && a->block_table && a->seq_lens, "null tensor pointer");
  LatAttnParams p = {};
  p.qs[0] = axis_stride(a->B, a->q_stride[0]);
  p.qs[1] = axis_stride(a->Sq, a->q_stride[1]);
  p.qs[2] = axis_stride(a->H, a->q_stride[2]);
  PITH_REQUIRE(aligned16(a->q) && aligned16(a->out) && aligned16(a->workspace) && p.qs[0] % 8 == 0 && p.qs[1] % 8 == 0 &&
                   p.qs[2] % 8 == 0,
               "q, out and workspace must be 16-byte aligned, q with strides that are multiples of 8 elements");
  PITH_REQUIRE(a->table_cols >= 0 && static_cast<int64_t>(a->table_cols) * a->cache.page_size < 2147483647 - 1024,
               "the block table covers too many keys");
  const int64_t rows = static_cast<int64_t>(a->Sq) * a->H;
  PITH_REQUIRE(rows < 2147483647 - 256, "too many query rows");
  const bool fp8 = a->cache.dtype == PITH_DTYPE_E4M3;
  const int nt = lat_rows(rows, fp8);
  const int64_t rt = (rows + nt - 1) / nt;
  PITH_REQUIRE(rt * a->B * (static_cast<int64_t>(a->table_cols) * a->cache.page_size / kBox + 2 + kMaxExtra) < 2147483647 - 1024,
               "too many query rows and keys for one call");
  if (int rc = require_sm100()) return rc;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  p.table = a->block_table; p.lens = a->seq_lens; p.qlens = a->query_lens; p.tree = a->tree_mask;
  p.scale = a->cache.scale; p.status = a->status;
  p.B = a->B; p.Sq = a->Sq; p.H = a->H; p.R = static_cast<int>(rows); p.RT = static_cast<int>(rt);
  p.pages = a->cache.pages; p.page_size = a->cache.page_size;
  p.max_keys = a->table_cols * a->cache.page_size;
  p.by_h = FastDiv(p.H);
  p.by_rt = FastDiv(p.RT);
  p.by_page = FastDiv(p.page_size);
  p.tile_pages = kTile / p.page_size;
  p.tile_rows = kTile % p.page_size;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.table_stride = a->table_stride;
  for (int i = 0; i < 2; ++i) { p.tree_stride[i] = a->tree_stride[i]; p.scale_stride[i] = a->cache.scale_stride[i]; }
  LatPlan plan;
  if (int rc = lat_plan(rt * a->B, p.max_keys, fp8, &plan)) return rc;
  const int ctas = plan.ctas;
  p.unit_log2 = plan.unit_log2;
  p.whole = p.max_keys <= (1 << plan.unit_log2);
  if (!p.whole) {
    PITH_REQUIRE(a->workspace, "null workspace");
    PITH_REQUIRE(a->workspace_bytes >= static_cast<size_t>(ctas) * 2 * nt * (kLat * 4 + 8) + static_cast<size_t>(ctas) * 16,
                 "workspace too small");
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    ws += static_cast<size_t>(ctas) * 2 * nt * kLat * 4;
    p.part_info = reinterpret_cast<int4*>(ws);
    ws += static_cast<size_t>(ctas) * 16;
    p.part_ml = reinterpret_cast<float2*>(ws);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp8) return nt == 16 ? launch_latent_attn<16, true>(a, p, ctas, st) : launch_latent_attn<32, true>(a, p, ctas, st);
  if (nt == 16) return launch_latent_attn<16, false>(a, p, ctas, st);
  if (nt == 32) return launch_latent_attn<32, false>(a, p, ctas, st);
  return launch_latent_attn<64, false>(a, p, ctas, st);
}
