// Attention over the quantised key/value cache for many query rows per kv head
// (chunks, prefixes): the fifth-generation tensor cores on keys and values that
// are turned back into bf16 on the way.
//
// The rows of a (sequence, kv head) are its G query heads of every query token,
// r = i G + head; an item is a block of 256 of them (two 128-row tiles, one per
// softmax group), a unit 128 keys (two pages, which need not be neighbours: the
// first tokens and the window's).  The units of all items make one line that is
// dealt out evenly to the persistent CTAs (kv_attention.cuh), so causal masks,
// windows and uneven lengths leave no SM waiting; an item cut by a CTA's border
// leaves fp32 sums that join_kernel adds.  Where an item has a few units at most
// (split == 0), items are dealt out whole, which spares the counting of all
// units before the first one and the second launch.  Warp roles:
//   warp 0       the CTA's segments (shares of items), for the other roles
//   warp 1       S issuer: S = Q_g K^T (128 x 128), unit by unit, group 0 then 1, into
//                three TMEM buffers in turn: it runs ahead of the softmax
//   warp 2       P.V issuer in the same order: O_g += P V (P from TMEM, where its S was;
//                V as the MN-major operand)
//   warps 4..11  codes to bf16: each takes 16 keys of the unit, copies their codes
//                and scales two units ahead (cp.async into a ring of its own) and
//                writes code * scale, exact in bf16, into the swizzled K and V
//                rings.  This is what the kernel adds to one over a bf16 cache; four
//                such warps took 2900 cycles a unit and held the others back.
//   warps 12..27 softmax: two threads per row, each 64 of a unit's 128 keys (one
//                page), which tell each other their maxima; they also bring the next
//                segment's queries (cp.async) and write a segment's rows out, after the
//                next one's first scores, which do not need O: so the last P.V is not
//                waited for by itself.  Sixteen warps, because one warp's chain of TMEM
//                loads, exponentials and packing, not any pipe, is what a unit waits
//                for: with one thread per row (eight warps) 1024 rows over 4 x 8192 keys
//                took 190 us.
// What bounds it.  A unit (256 rows x 128 keys) takes about 5000 SM cycles, and no
// pipe is full: the exponentials are 2048 of them on the MUFU (49 % busy), the tensor
// pipe 1200; 70 % of the issue slots are used, a third of them by waiting warps.  It
// is a row's chain: three TMEM loads that are each waited for, the maxima's swap, the
// exponentials, the store.  1024 rows over 4 caches of up to 8192 keys (15 / 5 heads, 4
// bits): 173 us, 461 TFLOP/s.  A block takes that time however many of its rows are
// there: 33 rows over 64 x 8000 keys (5 heads) 265 us, 128 rows 270, 150 rows 299 (8
// bits: 276, 284, 320).  One-unit
// items are one chain of latencies each, about 8000 cycles (queries, scores, maximum,
// exponentials, the last item's rows): 50 rows over each of 256 prefixes of up to 113
// keys 54 us (66 with the rows out before the next scores and all units dealt out); 50
// rows over 16 windows of 3729 keys 53 us.  Slower: an exponential token between the
// groups, exponentials partly on the FMA pipe, polling with a sleep, queries by TMA
// (whole query tokens per block leave a thirteenth block of 3072 rows) or by a warp of
// their own (one warp's copies take 8000 cycles a segment), rows out by the converting
// warps (61 us), the few-row kernel in blocks of 32 rows (177 us).
// A key that a row does not see must not reach it.  Its S is replaced by -inf;
// its value has the probability 0, and 0 times a value must be 0: slots past a
// sequence's length are written as zeros, and a value group whose scale is NaN
// (an input's NaN or infinity) is written as zeros and flagged, and the rows
// that see it are made NaN at the end.  A slot that no append wrote may hold a
// finite scale whose products leave bf16 (append writes none): they are held to
// its largest number.
#pragma once
#include "attention_tc.cuh"
#include "kv_attention.cuh"

namespace vla {
namespace kv {
namespace tc {

constexpr int BQ = 128;
constexpr int kRows = 2 * BQ;  // rows of an item
constexpr int kKeys = 128;     // keys of a unit
constexpr int kCodeWarps = 8, kSoft0 = 4 + kCodeWarps;  // converting warps; the first softmax warp
constexpr int kThreads = (kSoft0 + 16) * 32;
constexpr int kLaunchRegs = 72;  // 65536 / 896, rounded down to a multiple of 8
constexpr int kIssueRegs = 40;   // warps 0..3
constexpr int kCodeRegs = 56;    // warps 4..11
constexpr int kSoftRegs = 88;    // warps 12..27
static_assert(kIssueRegs + 2 * kCodeRegs + 4 * kSoftRegs == 7 * kLaunchRegs, "register split must equal the launch total");
constexpr int kRing = 3;    // K and V tiles
constexpr int kFlags = 4;   // flag sets: a softmax thread reads set j before S(j+1) may be issued
constexpr int TILE_BYTES = kKeys * HD * 2;
constexpr int kBuffers = 3;  // S and P of a tile (unit t, group g) in buffer (2 t + g) % 3
constexpr uint32_t O_COL0 = kBuffers * kKeys;
constexpr float kRescaleLog2 = 8.f;

// What a converting warp copies: a tile of 16 keys.
template <int BITS>
struct Raw {
  static constexpr int kCodes = Block<BITS>::kTileCodes;  // of the keys, or of the values
  static constexpr int kBytes = 2 * kCodes + 128;
  static constexpr int kStages = 3;
};

// Exponent field of a scale from which on a code (at most 8, or 128) times the
// scale may be 2^128 or more; NaN and the infinities (255) are above it.
template <int BITS>
constexpr uint32_t kBigScale = BITS == 4 ? 252u : 248u;

struct Flags {              // per page of a unit
  uint16_t nan[2][2][4];    // [page][value group][tile]: keys whose scale is NaN
  uint32_t absent[2][4];    // [page][tile]: not there (the same in a page's four)
};

// A CTA's share of an item, as warp 0 hands it to the other roles; one without units ends
// the CTA's work.
struct Segment {
  Span sp;
  int b, h, r0;        // sequence, kv head, first row
  int u0, n;           // units [u0, u0 + n)
  int whole;           // ... are all of the item's
  long long slot;      // of its part in the workspace, in rows
};
// Entries: one is written again when its rows are out.
constexpr int kSegments = 8;

template <int BITS>
struct Smem {
  uint8_t q[2][2][TILE_BYTES];  // [buffer][tile]
  uint8_t k[kRing][TILE_BYTES];
  uint8_t v[kRing][TILE_BYTES];
  uint8_t raw[kCodeWarps][Raw<BITS>::kStages][Raw<BITS>::kBytes];  // [warp]
  Flags flags[kFlags];
  Segment seg[kSegments];
  uint64_t seg_full[kSegments], seg_empty[kSegments];
  uint64_t q_full[2];  // [buffer]
  uint64_t k_full[kRing], k_empty[kRing];
  uint64_t v_full[kRing], v_empty[kRing];
  uint64_t s_full[kBuffers], s_empty[kBuffers];  // per buffer
  uint64_t p_full[2], pv_done[2];                // per group
  uint64_t drained[2];                           // S and P.V issuer, after an expired wait
  float swap[2][2][kRows];       // [turn][half of the keys]: maxima that a row's two threads tell each other
  float sum[2][2][kRows], top[2][kRows];  // [segment's parity]: what a segment's rows are finished with
  uint8_t nan[2][2][kRows];
  int scan[kThreads / 32];
  int group, left;
  uint32_t tmem_base;
  int abort;
};

// Pages [0, count) of an item's span as units of two.
__device__ __forceinline__ int units_of(const AttnParams& p, int group) {
  return (span_of(p, group / p.row_blocks, group % p.row_blocks * p.block, p.block).count + 1) / 2;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts8(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint32_t times(uint32_t x, uint32_t d2) { return as_u32(__hmul2(as_bf2(x), as_bf2(d2))); }
// x held to bf16's finite numbers (not for NaN)
__device__ __forceinline__ uint32_t finite(uint32_t x) {
  return as_u32(__hmax2(__hmin2(as_bf2(x), as_bf2(0x7F7F7F7Fu)), as_bf2(0xFF7FFF7Fu)));
}
// both halves: the low (high) half of x
__device__ __forceinline__ uint32_t lo2(uint32_t x) { return __byte_perm(x, x, 0x1010); }
__device__ __forceinline__ uint32_t hi2(uint32_t x) { return __byte_perm(x, x, 0x3232); }

// Which of 32 keys, the first at key0, a position sees.
__device__ __forceinline__ uint32_t seen32(int key0, int pos, int window, int sinks) {
  auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };  // keys 0 .. n - 1
  uint32_t m = below(pos - key0 + 1);
  if (window > 0) m &= ~below(pos - window + 1 - key0) | below(sinks - key0);
  return m;
}

// A tile's codes to rows [r0, r0 + 16) of a K and a V tile.
template <int BITS>
__device__ __forceinline__ void convert(uint32_t raw, uint32_t kt, uint32_t vt, int r0, int live, bool clean,
                                        uint32_t mask, int lane) {
  constexpr int C = Raw<BITS>::kCodes;
  const int g = lane >> 2, t = lane & 3;
  {
    const uint32_t sc = raw + 2 * C;
    // keys: tokens a and a + 2, 8 dims of either group
    const int a = 4 * (g >> 1) + (g & 1);
    uint4 d = lds16(sc + g * 16);
    const int row = r0 + a;
#pragma unroll
    for (int n = 0; n < 2; ++n) {  // odd g the other way round: eight lanes then touch all banks
      const int grp = n ^ (g & 1);
      uint32_t c[2][4];
      if (BITS == 4) {
        const uint4 w = lds16(raw + lane * 16);
        codes4(grp == 0 ? w.x : w.y, mask, c[0]);
        codes4(grp == 0 ? w.z : w.w, mask, c[1]);
      } else {
        const uint4 w = lds16(raw + grp * 512 + lane * 16);
        codes8(w.x, mask, c[0]);
        codes8(w.y, mask, c[0] + 2);
        codes8(w.z, mask, c[1]);
        codes8(w.w, mask, c[1] + 2);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t s = k == 0 ? d.x : d.z, s2 = grp == 0 ? lo2(s) : hi2(s);
        const int rr = row + 2 * k;
        sts16(kt + rr * 128 + (((grp * 4 + t) ^ (rr & 7)) << 4), times(c[k][0], s2), times(c[k][1], s2),
              times(c[k][2], s2), times(c[k][3], s2));
      }
    }
    // values: tokens 4q .. 4q + 3, 4 dims of either group
    const int q = lane >> 3, w8 = lane & 7;
    const uint4 sa = lds16(sc + q * 32), sb = lds16(sc + q * 32 + 16);
    const uint32_t vs[4] = {sa.y, sb.y, sa.w, sb.w};
    uint4 w0, w1;
    if (BITS == 4) {
      w0 = lds16(raw + C + lane * 16);
    } else {
      w0 = lds16(raw + C + lane * 16);
      w1 = lds16(raw + C + 512 + lane * 16);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int rr = r0 + 4 * q + r;
      uint32_t d0 = lo2(vs[r]), d1 = hi2(vs[r]);
      if (!clean) {  // past the end, or NaN (flagged)
        const bool past = 4 * q + r >= live;
        if (past || (d0 & 0x7F80u) == 0x7F80u) d0 = 0u;
        if (past || (d1 & 0x7F80u) == 0x7F80u) d1 = 0u;
      }
      uint32_t c[4];
      if (BITS == 4) {
        codes4(r == 0 ? w0.x : r == 1 ? w0.y : r == 2 ? w0.z : w0.w, mask, c);
      } else {
        codes8(r == 0 ? w0.x : r == 1 ? w0.y : r == 2 ? w0.z : w0.w, mask, c);
        codes8(r == 0 ? w1.x : r == 1 ? w1.y : r == 2 ? w1.z : w1.w, mask, c + 2);
      }
      const uint32_t at = vt + rr * 128 + (w8 & 1) * 8;
      sts8(at + (((w8 >> 1) ^ (rr & 7)) << 4), times(c[0], d0), times(c[1], d0));
      sts8(at + (((4 + (w8 >> 1)) ^ (rr & 7)) << 4), times(c[2], d1), times(c[3], d1));
    }
  }
}

__device__ __forceinline__ void tmem_start32(uint32_t a, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
// waits for the loads in flight; the registers pass through it, so no use moves above
__device__ __forceinline__ void tmem_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
        "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
        "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
        "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :: "memory");
}
__device__ __forceinline__ void tmem_put16(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int BITS>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  Smem<BITS>& sm = *reinterpret_cast<Smem<BITS>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = &sm.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.Lq * p.G, heads = p.c.kv_heads, groups = p.c.batch * p.row_blocks;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 16);
      mbar_init(&sm.p_full[i], 256);
      mbar_init(&sm.pv_done[i], 1);
      mbar_init(&sm.drained[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.s_empty[i], 1);
    }
    for (int s = 0; s < kSegments; ++s) {
      mbar_init(&sm.seg_full[s], 1);
      mbar_init(&sm.seg_empty[s], 16);
    }
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&sm.k_full[s], kCodeWarps);
      mbar_init(&sm.k_empty[s], 1);
      mbar_init(&sm.v_full[s], kCodeWarps);
      mbar_init(&sm.v_empty[s], 1);
    }
    sm.abort = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  pdl_prologue();

  // this CTA's share of the units, or (short caches) of the items
  int left, group0, at0;
  Deal d;
  if (p.split) {
    const int chunk = (groups + kThreads - 1) / kThreads;
    const int ga = min(groups, (int)threadIdx.x * chunk), gb = min(groups, ga + chunk);
    int mine = 0, before;
#pragma unroll 1
    for (int i = ga; i < gb; ++i) mine += units_of(p, i);
    d = deal_of(heads * block_scan<kThreads>(mine, &before, sm.scan), gridDim.x, 1);
    const int f0 = d.begin(blockIdx.x);
    left = (int)blockIdx.x < d.n ? d.begin(blockIdx.x + 1) - f0 : 0;
    if (left > 0 && f0 >= before * heads && f0 < (before + mine) * heads) {
      int at = f0 - before * heads, i = ga;
#pragma unroll 1
      for (;; ++i) {
        const int here = heads * units_of(p, i);
        if (at < here) break;
        at -= here;
      }
      sm.group = i;
      sm.left = at;
    }
    if (threadIdx.x == 0) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    group0 = sm.group;
    at0 = sm.left;
  } else {
    d = deal_of(groups * heads, gridDim.x, 1);
    const int f0 = d.begin(blockIdx.x);
    left = (int)blockIdx.x < d.n ? d.begin(blockIdx.x + 1) - f0 : 0;
    group0 = f0 / heads;
    at0 = f0 - group0 * heads;
  }
  // rows that see nothing belong to no unit
#pragma unroll 1
  for (int i = blockIdx.x; i < groups; i += gridDim.x) {
    const int b = i / p.row_blocks, r0 = i % p.row_blocks * p.block;
    if (units_of(p, i) > 0) continue;
#pragma unroll 1
    for (int x = threadIdx.x; x < heads * p.block * 8; x += kThreads) {
      const int hh = x / (p.block * 8), row = r0 + (x >> 3) % p.block, qi = row / p.G;
      if (row < rows)
        *reinterpret_cast<uint4*>(p.o + (long long)b * p.o_batch + (long long)qi * p.o_row +
                                  (long long)(hh * p.G + row - qi * p.G) * HD + (x & 7) * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  if (left > 0) {
    bool ok = true;
    int it = 0;  // segments
    auto segment = [&](int i) -> const Segment& {
      ok = mbar_wait_bounded(&sm.seg_full[i % kSegments], (i / kSegments) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      return sm.seg[i % kSegments];
    };
    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
      if (warp == 0) {
        // ---------------- segments ----------------
        int group = group0 - 1, h = heads, u0 = 0, units = 0;
        bool begin = true;
        Span sp;
#pragma unroll 1
        while (ok) {
          if (left > 0 && h == heads) {
            ++group;
            sp = span_of(p, group / p.row_blocks, group % p.row_blocks * p.block, p.block);
            units = (sp.count + 1) / 2;
            h = 0;
            if (begin) {
              h = p.split ? at0 / units : at0;
              u0 = p.split ? at0 - h * units : 0;
              begin = false;
            }
            if (units == 0) {
              left -= p.split ? 0 : heads - h;
              h = heads;
              continue;
            }
          }
          const int n = left <= 0 ? 0 : p.split ? min(units - u0, left) : units;
          left -= p.split ? n : 1;
          if (it >= kSegments)
            ok = mbar_wait_bounded(&sm.seg_empty[it % kSegments], ((it / kSegments) & 1) ^ 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) {
            Segment& sg = sm.seg[it % kSegments];
            sg.n = n;
            if (n > 0) {
              sg.sp = sp;
              sg.b = group / p.row_blocks;
              sg.h = h;
              sg.r0 = group % p.row_blocks * p.block;
              sg.u0 = u0;
              sg.whole = n == units;
              sg.slot = (2ll * blockIdx.x + (it > 0 ? 1 : 0)) * kRows;
            }
            mbar_arrive(&sm.seg_full[it % kSegments]);
            if (p.split && n > 0 && left == 0) record_cut(p, d, group, h, u0, u0 + n, units, it);
          }
          if (n == 0) break;
          u0 = 0;
          ++h;
          ++it;
        }
      } else if (warp == 1) {
        // ---------------- S issuer: group 0's tile, then group 1's ----------------
        constexpr uint32_t idesc_s = make_idesc_bf16(BQ, kKeys);
        int t = 0;
#pragma unroll 1
        for (;; ++it) {
          const Segment& sg = segment(it);
          const int n = sg.n, qb = it & 1;
          if (!ok || n == 0) break;
#pragma unroll 1
          for (int j = 0; ok && j < 2 * n; ++j) {
            const int tile = 2 * t + j, g = j & 1, buf = tile % kBuffers, sk = (tile >> 1) % kRing;
            if (j == 0) ok = mbar_wait_bounded(&sm.q_full[qb], (it >> 1) & 1, abort_flag);
            if (ok) ok = mbar_wait_bounded(&sm.k_full[sk], ((tile >> 1) / kRing) & 1, abort_flag);
            if (ok) ok = mbar_wait_bounded(&sm.s_empty[buf], ((tile / kBuffers) & 1) ^ 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);  // (lanes time their waits by themselves)
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t qdesc = make_sw128_desc(smem_u32(sm.q[qb][g]));
              const uint64_t kdesc = make_sw128_desc(smem_u32(sm.k[sk]));
#pragma unroll
              for (int k = 0; k < HD / 16; ++k)
                tc_mma_bf16(tmem + (uint32_t)(buf * kKeys), qdesc + 2 * k, kdesc + 2 * k, idesc_s, k > 0);
              tc_commit(&sm.s_full[buf]);
              if (g == 1) tc_commit(&sm.k_empty[sk]);
            }
            __syncwarp();
          }
          t += n;
        }
      } else if (warp == 2) {
        // ---------------- P.V issuer, in the same order ----------------
        constexpr uint32_t idesc_pv = make_idesc_bf16(BQ, HD) | (1u << 16);  // B (V) is MN-major
        int t = 0;
#pragma unroll 1
        for (;; ++it) {
          const int n = segment(it).n;
          if (!ok || n == 0) break;
#pragma unroll 1
          for (int j = 0; ok && j < 2 * n; ++j) {
            const int tile = 2 * t + j, g = j & 1, buf = tile % kBuffers, sv = (tile >> 1) % kRing;
            ok = mbar_wait_bounded(&sm.p_full[g], (uint32_t)(tile >> 1) & 1u, abort_flag);
            if (ok) ok = mbar_wait_bounded(&sm.v_full[sv], ((tile >> 1) / kRing) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t p_tmem = tmem + (uint32_t)(buf * kKeys), o_tmem = tmem + O_COL0 + (uint32_t)(g * HD);
              const uint32_t vbase = smem_u32(sm.v[sv]);
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)  // 16 keys; P of 32 keys lies where their S began
                attn_tc::tc_mma_bf16_ts(o_tmem, p_tmem + (uint32_t)((k >> 1) * 32 + (k & 1) * 8),
                                        attn_tc::make_sw128_mn_desc(vbase + (uint32_t)k * 2048u, 16384u), idesc_pv,
                                        (j > 1 || k > 0) ? 1u : 0u);
              tc_commit(&sm.pv_done[g]);
              tc_commit(&sm.s_empty[buf]);
              if (g == 1) tc_commit(&sm.v_empty[sv]);
            }
            __syncwarp();
          }
          t += n;
        }
      }
      if (!ok && (warp == 1 || warp == 2)) {  // products in flight end before the TMEM is freed (bounded)
        if (elect_one()) tc_commit(&sm.drained[warp - 1]);
        __syncwarp();
        mbar_wait_bounded(&sm.drained[warp - 1], 0, nullptr, 2000000ull);
      }
    } else if (warp < kSoft0) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCodeRegs));
      // ---------------- codes to bf16 ----------------
      using Rw = Raw<BITS>;
      const int w = warp - 4;  // keys [16 w, 16 w + 16) of a unit: tile w % 4 of page w / 4
      const uint32_t raw = smem_u32(sm.raw[w]);
      // step c copies unit c and converts unit c - kStages + 1, each with a segment of its own
      int ci = 0, cu = 0, cn = 0, cb = 0, ch = 0, csink = 0, cfirst = 0, ccount = 0;
      int u0 = 0, n = 0, j = 0, len = 0, sink = 0, first = 0;
      bool cmore = true;
      uint32_t there = 0;  // bit (stage): the page exists
#pragma unroll 1
      for (int c = 0; ok; ++c) {
        const bool there_now = (there >> ((c + 1) % Rw::kStages)) & 1u;  // of the unit to convert
        if (cn == 0 && cmore) {
          const Segment& sg = segment(ci++);
          if (!ok) break;
          cu = sg.u0;
          cn = sg.n;
          cb = sg.b;
          ch = sg.h;
          csink = sg.sp.sink;
          cfirst = sg.sp.first;
          ccount = sg.sp.count;
          cmore = cn > 0;
        }
        if (cn > 0) {
          const int st = c % Rw::kStages, u = 2 * cu + (w >> 2);
          bool have = false;
          if (u < ccount) {
            const int page = p.c.table[(long long)cb * p.c.table_ld + (u < csink ? u : cfirst + u - csink)];
            have = page >= 0 && page < p.c.pages;
            if (have) {
              const uint8_t* blk = p.c.pool + ((long long)page * heads + ch) * Block<BITS>::kBytes;
              const uint32_t dst = raw + st * Rw::kBytes + lane * 16;
              const uint8_t* src = blk + (w & 3) * Rw::kCodes + lane * 16;
#pragma unroll
              for (int i = 0; i < Rw::kCodes / 512; ++i) {
                copy16(dst + i * 512, src + i * 512);
                copy16(dst + Rw::kCodes + i * 512, src + Block<BITS>::kValues + i * 512);
              }
              if (lane < 8)
                copy16(dst + 2 * Rw::kCodes, blk + Block<BITS>::kScales + (w & 3) * 128 + lane * 16);
            } else {
              vla_record_range();
            }
          }
          there = have ? there | (1u << st) : there & ~(1u << st);
          ++cu;
          --cn;
        }
        copy_commit();
        const int t = c - (Rw::kStages - 1);
        if (t < 0) continue;
        if (j == n) {
          const Segment& sg = segment(it++);
          if (!ok) break;
          n = sg.n;
          if (n == 0) break;
          u0 = sg.u0;
          len = sg.sp.len;
          sink = sg.sp.sink;
          first = sg.sp.first;
          j = 0;
        }
        const int st = t % Rw::kStages, sr = t % kRing;
        const bool have = there_now;
        copy_wait<Rw::kStages - 1>();
        __syncwarp();
        ok = mbar_wait_bounded(&sm.k_empty[sr], ((t / kRing) & 1) ^ 1, abort_flag);
        if (ok) ok = mbar_wait_bounded(&sm.v_empty[sr], ((t / kRing) & 1) ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t kt = smem_u32(sm.k[sr]), vt = smem_u32(sm.v[sr]), from = raw + st * Rw::kBytes;
        const int u = 2 * (u0 + j) + (w >> 2), page = u < sink ? u : first + u - sink;
        int live = 0;  // of the 16 keys, those inside the sequence
        uint32_t n0 = 0u, n1 = 0u;
        if (have) {
          live = min(16, len - (page * kUnit + (w & 3) * 16));
          // key `lane`: token 4 q + b + 2 c at (2 q + b) * 16 + c * 8
          uint32_t s;
          asm volatile("ld.shared.u32 %0, [%1];"
                       : "=r"(s)
                       : "r"(from + 2 * Rw::kCodes + (2 * ((lane & 15) >> 2) + (lane & 1)) * 16 + ((lane >> 1) & 1) * 8 + 4));
          n0 = __ballot_sync(0xffffffffu, lane < live && (s & 0x7F80u) >= kBigScale<BITS> << 7);
          n1 = __ballot_sync(0xffffffffu, lane < live && (s & 0x7F800000u) >= kBigScale<BITS> << 23);
          convert<BITS>(from, kt, vt, w * 16, live, live == 16 && (n0 | n1) == 0u, p.mask, lane);
          if ((n0 | n1) != 0u) {  // rare: of these the NaN are flagged, the others' products held finite
            n0 = __ballot_sync(0xffffffffu, lane < live && (s & 0x7F80u) == 0x7F80u);
            n1 = __ballot_sync(0xffffffffu, lane < live && (s & 0x7F800000u) == 0x7F800000u);
            __syncwarp();  // the warp's rows are written
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
              const uint32_t at = vt + w * 2048 + i * 512 + lane * 16;
              const uint4 x = lds16(at);
              sts16(at, finite(x.x), finite(x.y), finite(x.z), finite(x.w));
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sts16(kt + w * 2048 + i * 512 + lane * 16, 0u, 0u, 0u, 0u);
            sts16(vt + w * 2048 + i * 512 + lane * 16, 0u, 0u, 0u, 0u);
          }
        }
        if (lane == 0) {
          Flags& f = sm.flags[t % kFlags];
          f.nan[w >> 2][0][w & 3] = (uint16_t)n0;
          f.nan[w >> 2][1][w & 3] = (uint16_t)n1;
          f.absent[w >> 2][w & 3] = have ? 0u : 1u;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.k_full[sr]);
          mbar_arrive(&sm.v_full[sr]);
        }
        ++j;
      }
      copy_wait<0>();
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
      // ---------------- softmax / output ----------------
      const int g = (warp - kSoft0) >> 3, hf = ((warp - kSoft0) >> 2) & 1, q = warp & 3;  // query tile, half of the keys, lane quarter
      const uint32_t lane_base = (uint32_t)(q * 32) << 16;
      const uint32_t s_adr0 = tmem + lane_base + (uint32_t)(hf * kUnit);
      const uint32_t o_adr = tmem + lane_base + O_COL0 + (uint32_t)(g * HD + hf * (HD / 2));
      int t = 0, turn = 0;
      // Tells the row's other thread v, returns what it tells.  The two warps meet
      // at a named barrier; one that gives up arrives there (below), so none is left waiting.
      const int at = g * BQ + q * 32 + lane;
      auto swap = [&](float v) {
        sm.swap[turn & 1][hf][at] = v;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + q) : "memory");
        float r;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(smem_u32(&sm.swap[turn & 1][hf ^ 1][at])));
        ++turn;
        ok = !__any_sync(0xffffffffu, *abort_flag);  // (raised before the other warp gave up)
        return r;
      };
      auto queries_there = [&]() {  // of the next segment
        copy_wait<0>();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[(it + 1) & 1]);
      };
      // 32 dims of segment i's rows, whose last P.V is done
      auto rows_out = [&](int i) {
        const Segment& sg = sm.seg[i % kSegments];
        const int row = sg.r0 + at, tok = row / p.G;
        if (row - lane < rows) {
          float o[HD / 2];
          tmem_ld32(o_adr, o);  // warp-collective: every lane loads
          const float l = sm.sum[i & 1][0][at] + sm.sum[i & 1][1][at];
          const bool nan = ((sm.nan[i & 1][0][at] | sm.nan[i & 1][1][at]) >> hf) & 1u;
          if (row < rows && sg.whole) {
            const bool zero = tok >= sg.sp.ql || (l == 0.f && !nan);
            const float inv = 1.f / l;
#pragma unroll
            for (int c = 0; c < HD / 2; ++c) o[c] = zero ? 0.f : nan ? __uint_as_float(0x7FC00000u) : o[c] * inv;
            bf16* out = p.o + (long long)sg.b * p.o_batch + (long long)tok * p.o_row +
                        (long long)(sg.h * p.G + row - tok * p.G) * HD + hf * (HD / 2);
#pragma unroll
            for (int c = 0; c < HD / 2; c += 8) *reinterpret_cast<uint4*>(out + c) = pack_bf16x8(o + c);
          } else if (row < rows) {
            const long long slot = sg.slot + at;
            float* part = p.part_o + slot * HD + hf * (HD / 2);
#pragma unroll
            for (int c = 0; c < HD / 2; c += 4)
              *reinterpret_cast<float4*>(part + c) =
                  nan ? make_float4(NAN, NAN, NAN, NAN) : make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
            if (hf == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(sm.top[i & 1][at], l);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.seg_empty[i % kSegments]);
      };
      const int tokens4 = 4 / p.G, heads4 = 4 - tokens4 * p.G;
      bool more = true;
#pragma unroll 1
      for (it = -1;; ++it) {  // (-1: only the first segment's queries)
        if (more) {
          // the next segment's queries to their buffer (S of the segment before, its last
          // reader, is done): each warp 16 rows, 4 rows an instruction
          const Segment& sg = segment(it + 1);
          if (!ok) break;
          more = sg.n > 0;
          if (more) {
            const int from = (hf * 4 + q) * 16 + (lane >> 3), qrow = sg.r0 + g * BQ + from;
            const uint32_t dst = smem_u32(sm.q[(it + 1) & 1][g]) + from * 128;
            int qi = qrow / p.G, head = qrow - qi * p.G;
            const bf16* src = p.q + (long long)sg.b * p.q_batch + (long long)sg.h * p.G * HD + (lane & 7) * 8;
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              const bool in = qrow + k < rows;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                               dst + k * 128 + (((lane & 7) ^ ((from + k) & 7)) << 4)),
                           "l"(in ? src + (long long)qi * p.q_row + head * HD : p.q), "r"(in ? 16 : 0)
                           : "memory");
              qi += tokens4;
              head += heads4;
              if (head >= p.G) {
                head -= p.G;
                ++qi;
              }
            }
            copy_commit();
          }
        }
        if (it < 0) {
          if (!more) break;
          queries_there();
          continue;
        }
        const Segment& sg = sm.seg[it % kSegments];
        const Span sp = sg.sp;
        const int u0 = sg.u0, n = sg.n, r0 = sg.r0, row = r0 + at;
        const int i = row / p.G;
        const bool none = i >= sp.ql;
        const int pos = row < rows && !none ? sp.pos(i, p.causal) : -1;
        const bool idle = n == 0 || row - lane >= rows;  // no row in this warp
        float m = -INFINITY, l = 0.f;
        uint32_t nan = 0;
#pragma unroll 1
        for (int j = 0; j < n || j == 0; ++j, ++t) {
          const int tile = 2 * t + g, buf = tile % kBuffers;
          if (n > 0) {
            ok = mbar_wait_bounded(&sm.s_full[buf], (uint32_t)(tile / kBuffers) & 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
          }
          if (!idle) {
            const uint32_t s_adr = s_adr0 + (uint32_t)(buf * kKeys);
            uint32_t r[32];
            tmem_start32(s_adr, r);
            const int pg = sp.unit(2 * (u0 + j) + hf);
            bool plain = (pg >= sp.open && pg < sp.shut) || pg < sp.sink_open;  // every row sees the page
            uint32_t vis0 = 0u, vis1 = 0u;  // else: the keys that this one sees
            {
              const uint32_t f = smem_u32(&sm.flags[t % kFlags]);
              const uint4 nn = lds16(f + 16 * hf);
              const bool absent = lds16(f + 32 + 16 * hf).x != 0u;
              plain = plain && !absent;
              if (!plain || (nn.x | nn.y | nn.z | nn.w) != 0u) {
                vis0 = absent ? 0u : seen32(pg * kUnit, pos, p.window, p.sinks);
                vis1 = absent ? 0u : seen32(pg * kUnit + 32, pos, p.window, p.sinks);
                if (((nn.x & vis0) | (nn.y & vis1)) != 0u) nan |= 1u;
                if (((nn.z & vis0) | (nn.w & vis1)) != 0u) nan |= 2u;
              }
            }
            auto mask = [&](uint32_t v) {
              if (!plain) {
#pragma unroll
                for (int c = 0; c < 32; ++c) r[c] = (v >> c) & 1u ? r[c] : 0xFF800000u;
              }
            };
            // the row's maximum over the unit, from both threads
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            auto top = [&]() {
#pragma unroll
              for (int c = 0; c < 32; c += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  mx4[e] = max3(mx4[e], __uint_as_float(r[c + e]), __uint_as_float(r[c + 4 + e]));
              }
            };
            tmem_wait32(r);
            mask(vis0);
            top();
            tmem_start32(s_adr + 32, r);
            tmem_wait32(r);
            mask(vis1);
            top();
            float mx = max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3])) * p.scale_log2;
            mx = fmaxf(mx, swap(mx));
            if (!ok) break;
            const bool grow = mx > m + kRescaleLog2;  // (from no maximum, always)
            if (__any_sync(0xffffffffu, grow)) {
              const float alpha = grow ? ex2(m - mx) : 1.f;
              if (grow) {
                m = mx;
                l *= alpha;
              }
              if (j > 0) {
                ok = mbar_wait_bounded(&sm.pv_done[g], (uint32_t)(t - 1) & 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 16) {
                  float o[16];
                  uint32_t u[16];
                  tmem_ld16(o_adr + c, o);
#pragma unroll
                  for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * alpha);
                  attn_tc::tmem_st16(o_adr + c, u);
                }
              }
            }
            // P = exp2(S - m), rounded to bf16, over the S of the same 32 keys
            const float mbase = m == -INFINITY ? 0.f : m;
            float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int qt = 1; qt >= 0; --qt) {
              uint32_t pk[16];
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                float x0, x1;
                attn_tc::fma2(__uint_as_float(r[c]), __uint_as_float(r[c + 1]), p.scale_log2, -mbase, x0, x1);
                x0 = ex2(x0);
                x1 = ex2(x1);
                attn_tc::add2(rs[c & 2], rs[(c & 2) + 1], x0, x1);
                pk[c >> 1] = pack_bf16x2(x0, x1);
              }
              tmem_put16(s_adr + 32 * qt, pk);
              if (qt == 1) {
                tmem_start32(s_adr, r);
                tmem_wait32(r);
                mask(vis0);
              }
            }
            tmem_put_wait();
            l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
          }
          if (t > 0) {  // P is announced in step with P.V, one phase at a time
            ok = mbar_wait_bounded(&sm.pv_done[g], (uint32_t)(t - 1) & 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (j == 0) {
              // the last segment's O, before this one's: its rows leave while their P.V and this
              // segment's scores would only have been waited for
              if (idle) swap(0.f);  // (else the maxima's: the other thread's sum is there)
              if (!ok) break;
              tc_fence_after();
              int last = it - 1;
              asm volatile("" : "+r"(last));  // keeps what rows_out derives from it out of the loop's registers
              rows_out(last);
            }
          }
          if (n == 0) break;
          tc_fence_before();
          mbar_arrive(&sm.p_full[g]);
        }
        if (!ok || n == 0) break;
        if (more) queries_there();
        sm.sum[it & 1][hf][at] = l;
        sm.nan[it & 1][hf][at] = (uint8_t)nan;
        if (hf == 0) sm.top[it & 1][at] = m;
      }
      if (!ok) {  // the queries in flight land; release the row's other warp
        copy_wait<0>();
        if (lane == 0) {
          if (!*abort_flag) vla_record_error(VLA_DERR_ATTN_TIMEOUT);
          *abort_flag = 1;
        }
        __syncwarp();
        asm volatile("bar.arrive %0, 64;" ::"r"(1 + g * 4 + q) : "memory");
      }
    }
    if (!ok && lane == 0) {
      if (!*abort_flag) vla_record_error(VLA_DERR_ATTN_TIMEOUT);
      *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int BITS>
constexpr int smem_bytes() {
  return (int)sizeof(Smem<BITS>) + 1024;
}

}  // namespace tc
}  // namespace kv
}  // namespace vla
