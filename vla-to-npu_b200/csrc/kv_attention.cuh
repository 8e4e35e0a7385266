// Attention over the quantised key/value cache (kvcache.cuh), head_dim 64, for
// few query rows per kv head: single tokens, short chunks.
//
//   O[r] = sum_j p_rj V[j] / sum_j p_rj,  p_rj = exp(scale q_r . K[j] - m_r)
//
// over the keys j that row r sees (position and window, below), m_r a running
// maximum.  The G = Hq / Hkv query heads of a kv head and its query tokens are
// stacked into rows r = i G + head, so a block of the cache is read once for all
// of them.  mma.m16n8k16 takes 16 KEYS (then 16 value dims) as its 16-row
// operand and 8 query rows as its 8 columns: S^T = K Q^T and O^T = V^T P^T, so
// few rows leave little of the tensor work unused, and the accumulator of S^T,
// packed to bf16 and transposed in 8 x 8 pieces (movmatrix), is P^T's operand.
// Scales never touch the elements: with s0, s1 the two groups' partial products,
// S = d0 s0 + d1 s1 per key in fp32, and P^T is multiplied by the value scales
// (fp32) before it is rounded to bf16.  Codes are finite whatever the memory
// holds, and p d is selected to 0 where a key is not seen, so an unwritten or
// masked slot's contents (NaN scales included) reach nothing.
//
// What bounds it.  The cache is read once: 72 bytes (4 bits) per key and kv head
// against 50 SM cycles for 16 keys at the measured copy rate.  16 keys cost a
// warp about 170 instructions, 88 of them on the integer pipe that issues every
// other cycle (masks and shifts 56, permutes, packing, maxima), so that pipe
// would allow 88 % of the copy rate; it is 58 % busy, the rest being dependent
// issue and the ends of the shares.  One token over 64 caches of up to 16001 keys
// (B200, 15 / 5 heads, 4 bits): 61 us, 3.8 TB/s, 0.58 of the measured copy; 96
// windows of 4096 keys in 8 bits with 32 / 8 heads: 87 us, 5.1 TB/s, 0.79 (in a
// graph; called one by one over caches of 2.5 GB in turn 91 to 96).
// More rows take two or four 8-row tiles (64 caches of 8000 keys, 5 kv heads, 4 / 8
// bits): 8 rows 54 / 72 us, 16 rows 78 / 90, 32 rows 124 / 132.  Four tiles in 4
// bits want more than the 255 registers that a thread has: 192 bytes spill (172 with
// the product taken twice; in 8 bits 0 and 12).
// Steps that led here, on the first of these: registers instead of the ring
// 84.6 us, ring 67.9 with one-instruction masks (89.9 with two), even shares
// 63.9, cuts joined from records 61.2.  Slower: shifts as multiplications on the
// other pipe (81), more resident warps (64.6), eight warps per CTA (63.8).
#pragma once
#include <type_traits>

#include "kvcache.cuh"

namespace vla {
namespace kv {

constexpr int kUnit = kPage;  // keys a warp takes at a time
constexpr int kHalf = kUnit / 2;

struct AttnParams {
  Cache c;
  const bf16* q;
  bf16* o;
  long long q_row, q_batch, o_row, o_batch;
  const int* lens;   // keys of each sequence
  const int* q_len;  // valid query tokens per sequence, or null: Lq
  int Lq, G;
  int causal, window, sinks;
  float scale_log2;
  uint32_t mask;     // code_mask<BITS>()
  int block, row_blocks;  // rows of a block, blocks per (sequence, kv head)
  int split;         // 1: all units dealt out to the CTAs evenly; 0: items whole (here a CTA each)
  float* part_o;     // split: [CTA][2][8 NT][64]
  float* part_ml;    //        [CTA][2][8 NT][2]
  int4* cut;         //        [CTA]: the item that starts in this CTA and goes on in others
};

// What a block of rows [r0, r0 + n) of one sequence sees: units (pages) [0, sink) and
// [first, last], numbered 0 .. count - 1.
struct Span {
  int len, ql;    // keys, valid query tokens
  int lo, hi;     // positions of the first and last row's token
  int sink, first, count;
  int open, shut, sink_open;  // units that every row sees whole: [open, shut) and [0, sink_open)
  __device__ __forceinline__ int unit(int u) const { return u < sink ? u : first + u - sink; }
  __device__ __forceinline__ int pos(int i, int causal) const { return causal ? len - ql + i : len - 1; }
};

__device__ __forceinline__ Span span_of(const AttnParams& p, int b, int r0, int n) {
  Span s;
  s.len = p.lens[b];
  const long long room = (long long)p.c.max_pages * kPage;
  if (s.len < 0 || s.len > room) {
    vla_record_range();
    s.len = s.len < 0 ? 0 : (int)room;
  }
  s.ql = p.q_len != nullptr ? max(0, min(p.Lq, p.q_len[b])) : p.Lq;
  const int i0 = r0 / p.G, i1 = min((r0 + n - 1) / p.G, s.ql - 1);
  s.lo = s.pos(i0, p.causal);
  s.hi = s.pos(i1, p.causal);
  s.sink = s.first = s.count = s.open = s.shut = s.sink_open = 0;
  if (i0 > i1 || s.hi < 0) return s;
  s.shut = max(0, s.lo + 1) / kUnit;
  if (p.window > 0) {
    s.open = (max(0, s.hi - p.window + 1) + kUnit - 1) / kUnit;
    s.sink_open = min(p.sinks / kUnit, s.shut);
    s.first = max(0, s.lo - p.window + 1) / kUnit;
    s.sink = min((p.sinks + kUnit - 1) / kUnit, s.first);
  }
  s.count = s.sink + s.hi / kUnit - s.first + 1;
  return s;
}

// D = A B + C with C and D apart, so that a start value need not be copied.
__device__ __forceinline__ void mma16n8(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float c0, float c1,
                                        float c2, float c3) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma16n8(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  mma16n8(d, a, b0, b1, d[0], d[1], d[2], d[3]);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Pages on their way through shared memory, one ring per warp; a stage is a page
// in 4 bits and half of one in 8.  Keys and scales keep their order (a lane's 16
// bytes lie at lane order); the 128-byte rows of the values (4 tokens) are 160
// bytes apart, so that the eight lanes of a 16-byte access, 2 words of 4 rows,
// touch all banks.
template <int BITS>
struct Ring {
  static constexpr int kSteps = BITS == 4 ? 1 : 2;  // stages of a page
  static constexpr int kTiles = 4 / kSteps;
  static constexpr int kChunks = kTiles * BITS / 4;  // 512-byte pieces of a stage's keys (or values)
  static constexpr int kVOff = kChunks * 512;
  static constexpr int kSOff = kVOff + kChunks * 640;
  static constexpr int kStage = kSOff + kTiles * 128;  // 5120 or 4864 bytes
  static constexpr int kStages = 2;
  static constexpr int kWarpBytes = kStage * kStages;
};

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

template <int BITS>
__device__ __forceinline__ void copy_stage(uint32_t stage, const uint8_t* blk, int step, int lane) {
  using B = Block<BITS>;
  using Rg = Ring<BITS>;
  const uint8_t* src = blk + step * (Rg::kChunks * 512) + lane * 16;
  const uint32_t vdst = stage + Rg::kVOff + (lane >> 3) * 160 + (lane & 7) * 16;
#pragma unroll
  for (int i = 0; i < Rg::kChunks; ++i) {
    copy16(stage + i * 512 + lane * 16, src + i * 512);
    copy16(vdst + i * 640, src + B::kValues + i * 512);
  }
  if (Rg::kTiles == 4 || lane < 16)
    copy16(stage + Rg::kSOff + lane * 16, blk + B::kScales + step * (Rg::kTiles * 128) + lane * 16);
}

// The lane's operand registers of one tile's keys and one group of dims:
// a[k-step][4] (rows g, g + 8; dims pairs).  4-bit codes stay 136 too large
// (128 + n instead of code = n - 8): the product starts from -136 sum(q)
// instead, which spares the subtractions; the sums' rounding, 2^-24 of
// 136 |sum q|, stays far below bf16's 2^-8 in the probabilities.
template <int BITS>
__device__ __forceinline__ void key_operand(const uint4* c, int grp, uint32_t mask, uint32_t (*a)[4]) {
  uint32_t lo[4], hi[4];  // token 4q+b (row g), token 4q+b+2 (row g + 8)
  if (BITS == 4) {
    const uint32_t wl = grp == 0 ? c[0].x : c[0].y, wh = grp == 0 ? c[0].z : c[0].w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = lop_and_or(wl >> (4 * i), mask, 0x43004300u);
      hi[i] = lop_and_or(wh >> (4 * i), mask, 0x43004300u);
    }
  } else {
    const uint4 w = c[grp];
    codes8(w.x, mask, lo);
    codes8(w.y, mask, lo + 2);
    codes8(w.z, mask, hi);
    codes8(w.w, mask, hi + 2);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    a[s][0] = lo[2 * s];
    a[s][1] = hi[2 * s];
    a[s][2] = lo[2 * s + 1];
    a[s][3] = hi[2 * s + 1];
  }
}

// The lane's operand registers of one tile's values, group grp: two 16-dim
// pieces m (rows: dims 4g + 2m and 4g + 2m + 1; columns: tokens 4t .. 4t+3).
template <int BITS>
__device__ __forceinline__ void value_operand(const uint4* c, int grp, uint32_t mask, uint32_t (*a)[4]) {
  const uint4 w = c[BITS == 4 ? 0 : grp];
  const uint32_t e01 = __byte_perm(w.x, w.y, 0x5410), o01 = __byte_perm(w.x, w.y, 0x7632);
  const uint32_t e23 = __byte_perm(w.z, w.w, 0x5410), o23 = __byte_perm(w.z, w.w, 0x7632);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (BITS == 4) {
      const int sh = 8 * grp + 4 * m;
      a[m][0] = as_u32(__hsub2(as_bf2(lop_and_or(e01 >> sh, mask, 0x43004300u)), as_bf2(0x43084308u)));
      a[m][1] = as_u32(__hsub2(as_bf2(lop_and_or(o01 >> sh, mask, 0x43004300u)), as_bf2(0x43084308u)));
      a[m][2] = as_u32(__hsub2(as_bf2(lop_and_or(e23 >> sh, mask, 0x43004300u)), as_bf2(0x43084308u)));
      a[m][3] = as_u32(__hsub2(as_bf2(lop_and_or(o23 >> sh, mask, 0x43004300u)), as_bf2(0x43084308u)));
    }
  }
  if (BITS == 8) {
    uint32_t x[4][2];
    codes8(e01, mask, x[0]);
    codes8(o01, mask, x[1]);
    codes8(e23, mask, x[2]);
    codes8(o23, mask, x[3]);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[m][i] = x[i][m];
    }
  }
}

constexpr int kWarps = 4;
template <int BITS, int NT>
constexpr int attend_smem() {
  const int rings = kWarps * Ring<BITS>::kWarpBytes, join = kWarps * 8 * NT * (HD + 4 + 2) * (int)sizeof(float);
  return rings > join ? rings : join;
}

// Groups are blocks of rows of a sequence (b, rb), items a group's kv heads; the
// units of all items in order, group by group and head by head, make one line.
// With `split` the line is cut into n shares that differ by one unit at most, so
// lengths however uneven leave no CTA waiting for another; n is the grid, or
// fewer when that would leave CTAs less than `least` units.  (Fewer than 2^31
// units: the host checks.)
struct Deal {
  int n, share, extra;  // the first `extra` shares have one unit more
  __device__ __forceinline__ int begin(int c) const { return c * share + min(c, extra); }
  __device__ __forceinline__ int owner(int unit) const {
    const int long_ones = extra * (share + 1);
    return unit < long_ones ? unit / (share + 1) : extra + (unit - long_ones) / share;
  }
};
__device__ __forceinline__ Deal deal_of(int total, int ctas, int least) {
  Deal d;
  d.n = max(1, min(ctas, (total + least - 1) / least));
  d.share = total / d.n;
  d.extra = total - d.share * d.n;
  return d;
}

// The sum of all threads' values; *before: of the threads below.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* before, int* shared) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int run = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, d);
    if (lane >= d) run += up;
  }
  if (lane == 31) shared[warp] = run;
  __syncthreads();
  int base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) base += shared[w];
    total += shared[w];
  }
  *before = base + run - v;
  return total;
}

// What CTA c's share ends with, for join_kernel: group, kv head, slot of the first
// part, number of parts (0: its last item ends with the share or started before).
__device__ __forceinline__ void record_cut(const AttnParams& p, const Deal& d, int group, int h, int u0, int u1,
                                           int units, int segment) {
  const int c = blockIdx.x;
  if (u1 < units)
    p.cut[c] = u0 == 0 ? make_int4(group, h, 2 * c + (segment > 0 ? 1 : 0),
                                   d.owner(d.begin(c + 1) - u1 + units - 1) - c + 1)
                       : make_int4(0, 0, 0, 0);
}

// A CTA's warps take the units of an item (or of its share of one) in turn, each
// with its own running maximum, sum and output, which are joined in shared memory
// at the item's end.  A warp copies pages into its own ring ahead of its
// computation (cp.async; no warp waits for another).
// TWICE: P^T goes through the product as the sum of two bf16 numbers, which takes its
// rounding (2^-8 of each term, as much as the output's own) out of the result.
// Used where the keys are few: there one of them often outweighs the rest, its
// rounding does not average out, and the call costs its launch; over long caches
// it would cost a tenth of the time.
template <int BITS, int NT, bool TWICE>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(AttnParams p) {
  pdl_prologue();
  constexpr int R = 8 * NT, kThreads = kWarps * 32;
  using Rg = Ring<BITS>;
  extern __shared__ __align__(128) uint8_t smem[];  // the rings; after an item's loop the warps' results
  __shared__ int s_scan[kWarps];
  __shared__ int s_group, s_left;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rows = p.Lq * p.G, heads = p.c.kv_heads, groups = p.c.batch * p.row_blocks;

  // where this CTA starts, and how many units it takes
  int group, h, u0, left;
  Deal d{};
  if (p.split) {
    const int chunk = (groups + kThreads - 1) / kThreads;
    const int ga = min(groups, (int)threadIdx.x * chunk), gb = min(groups, ga + chunk);
    int mine = 0, before;
    for (int i = ga; i < gb; ++i) mine += span_of(p, i / p.row_blocks, i % p.row_blocks * R, R).count;
    d = deal_of(heads * block_scan<kThreads>(mine, &before, s_scan), gridDim.x, kWarps);
    const int f0 = d.begin(blockIdx.x);
    left = (int)blockIdx.x < d.n ? d.begin(blockIdx.x + 1) - f0 : 0;
    if (left > 0 && f0 >= before * heads && f0 < (before + mine) * heads) {  // one thread's groups hold it
      int at = f0 - before * heads;
      int i = ga;
      for (;; ++i) {
        const int here = heads * span_of(p, i / p.row_blocks, i % p.row_blocks * R, R).count;
        if (at < here) break;
        at -= here;
      }
      s_group = i;
      s_left = at;
    }
    // rows that see nothing belong to no unit
    for (int i = blockIdx.x; i < groups; i += gridDim.x) {
      const int b = i / p.row_blocks, r0 = i % p.row_blocks * R;
      if (span_of(p, b, r0, R).count > 0) continue;
      for (int x = threadIdx.x; x < heads * R * 8; x += kThreads) {
        const int hh = x / (R * 8), row = r0 + (x >> 3) % R, qi = row / p.G;
        if (row < rows)
          *reinterpret_cast<uint4*>(p.o + (long long)b * p.o_batch + (long long)qi * p.o_row +
                                    (long long)(hh * p.G + row - qi * p.G) * HD + (x & 7) * 8) = make_uint4(0, 0, 0, 0);
      }
    }
    if (threadIdx.x == 0) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (left == 0) return;
    __syncthreads();
    group = s_group;
    const int count = span_of(p, group / p.row_blocks, group % p.row_blocks * R, R).count;
    h = s_left / count;
    u0 = s_left - h * count;
  } else {
    group = blockIdx.x / heads;
    h = blockIdx.x - group * heads;
    u0 = 0;
    left = 0x7FFFFFFF;
  }

  for (int segment = 0; left > 0; ++segment) {
  const int b = group / p.row_blocks, r0 = group % p.row_blocks * R;
  const Span sp = span_of(p, b, r0, R);
  const int u1 = min(sp.count - u0, left) + u0;

  // the units' pages
  const int* table = p.c.table + (long long)b * p.c.table_ld;
  auto page_of = [&](int u) { return u < u1 ? table[sp.unit(u)] : 0; };  // slots lie inside the table (span_of)
  auto block = [&](int u, int page) -> const uint8_t* {
    if (u >= u1) return nullptr;
    if (page < 0 || page >= p.c.pages) {
      vla_record_range();
      return nullptr;
    }
    return p.c.pool + ((long long)page * heads + h) * Block<BITS>::kBytes;
  };
  const int steps = u0 + warp < u1 ? Rg::kSteps * ((u1 - u0 - warp + kWarps - 1) / kWarps) : 0;
  const uint32_t ring = smem_u32(smem) + warp * Rg::kWarpBytes;
  int iu = u0 + warp, page = page_of(iu), next = 0, put = 0;  // copies: unit, page number, step, stage
  const uint8_t* blk = nullptr;
  uint32_t valid = 0;  // stages that hold (a part of) a page that exists
  auto issue = [&]() {
    if (next < steps) {
      if (Rg::kSteps == 1 || (next & 1) == 0) {
        blk = block(iu, page);
        iu += kWarps;
        page = page_of(iu);
      }
      valid = blk ? valid | (1u << put) : valid & ~(1u << put);
      if (blk) copy_stage<BITS>(ring + put * Rg::kStage, blk, next % Rg::kSteps, lane);
    }
    copy_commit();
    ++next;
    put = put == Rg::kStages - 1 ? 0 : put + 1;
  };
#pragma unroll
  for (int i = 0; i < Rg::kStages - 1; ++i) issue();

  // query operand: column g of n-tile j is row r0 + 8j + g, dims 32 grp + 8t .. + 7
  uint32_t qf[NT][2][4];
  int pos[NT][2];  // positions of the accumulator's columns 2t, 2t + 1
  float2 init[NT][2];  // what the columns' partial products start from
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = r0 + 8 * j + g;
    const int i = r / p.G, head = h * p.G + r - i * p.G;
#pragma unroll
    for (int grp = 0; grp < 2; ++grp) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows)
        x = ld_stream(p.q + (long long)b * p.q_batch + (long long)i * p.q_row + (long long)head * HD + grp * 32 + t * 8);
      qf[j][grp][0] = x.x;
      qf[j][grp][1] = x.y;
      qf[j][grp][2] = x.z;
      qf[j][grp][3] = x.w;
      init[j][grp] = make_float2(0.f, 0.f);
      if (BITS == 4) {
        float f[8];
        unpack_bf16x8(x, f);
        float sum = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        init[j][grp].x = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t);
        init[j][grp].y = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int rc = r0 + 8 * j + 2 * t + c, ic = rc / p.G;
      pos[j][c] = rc < rows && ic < sp.ql ? sp.pos(ic, p.causal) : -1;
    }
  }

  float o[NT][4][4];
  float m[NT][2];       // running maxima of the columns (raw products)
  float2 l[NT], ms[NT]; // sums of the lane's keys; -m * scale log2(e), 0 while there is no maximum
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    m[j][0] = m[j][1] = -INFINITY;
    l[j] = ms[j] = make_float2(0.f, 0.f);
  }
  // the maximum moves in steps above 2^8 only (of raw products; finite also for a scale near 0)
  const float grow = fminf(8.f / p.scale_log2, 0x1.fffffep127f);
  const uint32_t mask = p.mask;
  const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);

  auto compute = [&](uint32_t stage, int half, int key0, auto masked) {  // 32 keys
    constexpr bool MASK = decltype(masked)::value;
    const uint32_t ka = stage + half * (BITS * 256) + lane * 16;
    const uint32_t va = stage + Rg::kVOff + half * (BITS * 320) + t * 160 + g * 16;
    const uint32_t sa = stage + Rg::kSOff + half * 256 + g * 16;
    uint4 sc[2];
    sc[0] = lds16(sa);
    sc[1] = lds16(sa + 128);
    float2 s[2][NT][2];  // [tile][n-tile][key g or g + 8] over the columns 2t, 2t + 1
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s0[NT][4], s1[NT][4];
      uint32_t a[2][4];
      uint4 kc[BITS / 4];
#pragma unroll
      for (int c = 0; c < BITS / 4; ++c) kc[c] = lds16(ka + (i * (BITS / 4) + c) * 512);
      key_operand<BITS>(kc, 0, mask, a);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma16n8(s0[j], a[0], qf[j][0][0], qf[j][0][1], init[j][0].x, init[j][0].y, init[j][0].x, init[j][0].y);
        mma16n8(s0[j], a[1], qf[j][0][2], qf[j][0][3]);
      }
      key_operand<BITS>(kc, 1, mask, a);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma16n8(s1[j], a[0], qf[j][1][0], qf[j][1][1], init[j][1].x, init[j][1].y, init[j][1].x, init[j][1].y);
        mma16n8(s1[j], a[1], qf[j][1][2], qf[j][1][3]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t d = k == 0 ? sc[i].x : sc[i].z;
        const float d0 = __uint_as_float(d << 16), d1 = __uint_as_float(d & 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < NT; ++j)
          s[i][j][k] = __ffma2_rn(make_float2(s0[j][2 * k], s0[j][2 * k + 1]), make_float2(d0, d0),
                                  __fmul2_rn(make_float2(s1[j][2 * k], s1[j][2 * k + 1]), make_float2(d1, d1)));
      }
    }
    uint32_t hidden[NT];
    if (MASK) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        hidden[j] = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = e >> 2, k = (e >> 1) & 1, c = e & 1;
          const int key = key0 + i * 16 + 4 * (g >> 1) + (g & 1) + 2 * k, at = pos[j][c];
          if (key > at || (p.window > 0 && key <= at - p.window && key >= p.sinks)) {
            hidden[j] |= 1u << e;
            (c == 0 ? s[i][j][k].x : s[i][j][k].y) = -INFINITY;
          }
        }
      }
    }
    bool moves = false;
    float2 top[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      top[j].x = max3(s[0][j][0].x, s[0][j][1].x, fmaxf(s[1][j][0].x, s[1][j][1].x));
      top[j].y = max3(s[0][j][0].y, s[0][j][1].y, fmaxf(s[1][j][0].y, s[1][j][1].y));
      // (from no maximum, -inf + grow is -inf and any score moves it)
      moves |= top[j].x > m[j][0] + grow || top[j].y > m[j][1] + grow;
    }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float tp = c == 0 ? top[j].x : top[j].y;
          tp = fmaxf(tp, __shfl_xor_sync(0xffffffffu, tp, 4));
          tp = fmaxf(tp, __shfl_xor_sync(0xffffffffu, tp, 8));
          tp = fmaxf(tp, __shfl_xor_sync(0xffffffffu, tp, 16));
          const float to = fmaxf(m[j][c], tp);
          const float f = to == m[j][c] ? 1.f : ex2((m[j][c] - to) * p.scale_log2);
          m[j][c] = to;
          const float neg = to == -INFINITY ? 0.f : -to * p.scale_log2;
          if (c == 0) {
            ms[j].x = neg;
            l[j].x *= f;
          } else {
            ms[j].y = neg;
            l[j].y *= f;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[j][i][c] *= f;
            o[j][i][c + 2] *= f;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint4 vc[BITS / 4];
#pragma unroll
      for (int c = 0; c < BITS / 4; ++c) vc[c] = lds16(va + (i * (BITS / 4) + c) * 640);
      uint32_t pt[NT][2][2], rest[NT][2][2];  // P^T operand [n-tile][group][key half], and what it lost
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t d = k == 0 ? sc[i].y : sc[i].w;
        const float d0 = __uint_as_float(d << 16), d1 = __uint_as_float(d & 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float2 e = __ffma2_rn(s[i][j][k], sl2, ms[j]);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          l[j] = __fadd2_rn(l[j], e);
          float2 x0 = __fmul2_rn(e, make_float2(d0, d0)), x1 = __fmul2_rn(e, make_float2(d1, d1));
          if (MASK) {  // 0 times a scale that is NaN
            if ((hidden[j] >> (4 * i + 2 * k)) & 1u) x0.x = x1.x = 0.f;
            if ((hidden[j] >> (4 * i + 2 * k)) & 2u) x0.y = x1.y = 0.f;
          }
          // P^T with its value scales, rounded to bf16
          const uint32_t h0 = pack_bf16x2(x0.x, x0.y), h1 = pack_bf16x2(x1.x, x1.y);
          pt[j][0][k] = transpose8(h0);
          pt[j][1][k] = transpose8(h1);
          if (TWICE) {
            rest[j][0][k] = transpose8(pack_bf16x2(x0.x - __uint_as_float(h0 << 16), x0.y - __uint_as_float(h0 & 0xFFFF0000u)));
            rest[j][1][k] = transpose8(pack_bf16x2(x1.x - __uint_as_float(h1 << 16), x1.y - __uint_as_float(h1 & 0xFFFF0000u)));
          }
        }
      }
#pragma unroll
      for (int grp = 0; grp < 2; ++grp) {
        uint32_t a[2][4];
        value_operand<BITS>(vc, grp, mask, a);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma16n8(o[j][2 * grp], a[0], pt[j][grp][0], pt[j][grp][1]);
          mma16n8(o[j][2 * grp + 1], a[1], pt[j][grp][0], pt[j][grp][1]);
          if (TWICE) {
            mma16n8(o[j][2 * grp], a[0], rest[j][grp][0], rest[j][grp][1]);
            mma16n8(o[j][2 * grp + 1], a[1], rest[j][grp][0], rest[j][grp][1]);
          }
        }
      }
    }
  };

  int get = 0;
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    issue();
    copy_wait<Rg::kStages - 1>();
    __syncwarp();
    const int un = sp.unit(u0 + warp + i / Rg::kSteps * kWarps);
    if ((valid >> get) & 1u) {
      const uint32_t stage = ring + get * Rg::kStage;
      int key0 = un * kUnit + i % Rg::kSteps * kHalf;
      if ((un >= sp.open && un < sp.shut) || un < sp.sink_open) {
#pragma unroll
        for (int half = 0; half < 2 / Rg::kSteps; ++half) compute(stage, half, key0 + half * kHalf, std::false_type());
      } else {
#pragma unroll 1
        for (int half = 0; half < 2 / Rg::kSteps; ++half, key0 += kHalf)
          if (key0 <= sp.hi) compute(stage, half, key0, std::true_type());
      }
    }
    __syncwarp();
    get = get == Rg::kStages - 1 ? 0 : get + 1;
  }
  copy_wait<0>();
  __syncthreads();  // the rings' memory is free
  float(*sO)[R][HD + 4] = reinterpret_cast<float(*)[R][HD + 4]>(smem);
  float(*sM)[R] = reinterpret_cast<float(*)[R]>(smem + sizeof(float) * kWarps * R * (HD + 4));
  float(*sL)[R] = sM + kWarps;

  // join the warps: columns 2t, 2t+1 of n-tile j are rows 8j + 2t (+ 1); piece
  // 2 grp + n holds dims 32 grp + 4g + 2n and that + 1
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = c == 0 ? l[j].x : l[j].y;
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int r = 8 * j + 2 * t + c;
      if (g == 0) {
        sM[warp][r] = m[j][c];
        sL[warp][r] = sum;
      }
#pragma unroll
      for (int grp = 0; grp < 2; ++grp)
        *reinterpret_cast<float4*>(&sO[warp][r][32 * grp + 4 * g]) =
            make_float4(o[j][2 * grp][c], o[j][2 * grp][c + 2], o[j][2 * grp + 1][c], o[j][2 * grp + 1][c + 2]);
    }
  }
  __syncthreads();
  const bool whole = u0 == 0 && u1 == sp.count;
  const long long slot = 2ll * blockIdx.x + (segment > 0 ? 1 : 0);  // a CTA has at most two items in part: its first and last
  for (int y = threadIdx.x; y < R * 8; y += kWarps * 32) {
    const int r = y >> 3, d8 = (y & 7) * 8, row = r0 + r;
    if (row >= rows) continue;
    float top = sM[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sM[w][r]);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      // without a maximum the sum is 0, or NaN where every score of the warp is
      const float f = sM[w][r] == -INFINITY ? 0.f : ex2((sM[w][r] - top) * p.scale_log2);
      sum += sM[w][r] == -INFINITY ? sL[w][r] : f * sL[w][r];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f * sO[w][r][d8 + e];
    }
    if (whole) {
      const int i = row / p.G, head = h * p.G + row - i * p.G;
      const bool empty = i >= sp.ql || sum == 0.f;
      const float inv = empty ? 0.f : 1.f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = empty ? 0.f : acc[e] * inv;
      *reinterpret_cast<uint4*>(p.o + (long long)b * p.o_batch + (long long)i * p.o_row + (long long)head * HD + d8) =
          pack_bf16x8(acc);
    } else {
      float4* dst = reinterpret_cast<float4*>(p.part_o + (slot * R + r) * HD + d8);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (d8 == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * R + r) * 2) = make_float2(top, sum);
    }
  }
  if (!p.split) return;
  if (threadIdx.x == 0) record_cut(p, d, group, h, u0, u1, sp.count, segment);
  left -= u1 - u0;
  if (left > 0) {  // the next item that has units
    u0 = 0;
    if (++h == heads) {
      h = 0;
      do ++group;
      while (span_of(p, group / p.row_blocks, group % p.row_blocks * R, R).count == 0);
    }
    __syncthreads();  // the results' memory is the next item's ring
  }
  }
}

// Joins the parts of cut items, in the order of their CTAs: kWarpsPerRow warps per
// row share the parts, two dims per lane.  blockIdx: (slice of the rows, CTA).
constexpr int kJoinWarps = 8;
template <int R, int WPR>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(AttnParams p, float to_log2) {
  pdl_prologue();
  __shared__ float sO[kJoinWarps][HD];
  __shared__ float sL[kJoinWarps];
  const int4 cut = p.cut[blockIdx.y];
  const int n = cut.w;
  if (n == 0) return;
  const int b = cut.x / p.row_blocks, h = cut.y, r0 = cut.x % p.row_blocks * p.block;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x * (kJoinWarps / WPR) + warp / WPR, row = r0 + r;
  const bool there = r < p.block && row < p.Lq * p.G;
  // a part is its CTA's first item, but the first part may be its CTA's last
  auto slot = [&](int y) { return (long long)(y == 0 ? cut.z : 2 * ((int)blockIdx.y + y)) * R + r; };
  float sum = 0.f, a0 = 0.f, a1 = 0.f;
  if (there) {
    float top = -INFINITY;
    for (int y = lane; y < n; y += 32) top = fmaxf(top, p.part_ml[slot(y) * 2]);
    top = warp_max(top);
#pragma unroll 4
    for (int y = warp % WPR; y < n; y += WPR) {
      const float2 v = *reinterpret_cast<const float2*>(p.part_o + slot(y) * HD + 2 * lane);
      const float2 w = *reinterpret_cast<const float2*>(p.part_ml + slot(y) * 2);
      const float f = w.x == -INFINITY ? 0.f : ex2((w.x - top) * to_log2);
      sum += w.x == -INFINITY ? w.y : f * w.y;
      a0 += f * v.x;
      a1 += f * v.y;
    }
  }
  if (WPR > 1) {
    sO[warp][2 * lane] = a0;
    sO[warp][2 * lane + 1] = a1;
    if (lane == 0) sL[warp] = sum;
    __syncthreads();
    if (warp % WPR != 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      sum += sL[warp + w];
      a0 += sO[warp + w][2 * lane];
      a1 += sO[warp + w][2 * lane + 1];
    }
  }
  if (!there) return;
  const int i = row / p.G, head = h * p.G + row - i * p.G;
  const bool empty = (p.q_len != nullptr && i >= p.q_len[b]) || sum == 0.f;
  const float inv = empty ? 0.f : 1.f / sum;
  *reinterpret_cast<uint32_t*>(p.o + (long long)b * p.o_batch + (long long)i * p.o_row + (long long)head * HD +
                               2 * lane) = empty ? 0u : pack_bf16x2(a0 * inv, a1 * inv);
}

}  // namespace kv
}  // namespace vla
