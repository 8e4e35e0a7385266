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
// leaves fp32 sums that join_kernel adds.  Warp roles:
//   warp 0       the CTA's segments (shares of items), for the other roles
//   warps 1, 2   S issuers, one per group: S_g = Q_g K^T (128 x 128 into TMEM)
//   warp 3       P.V issuer: O_g += P_g V (P from TMEM, V as the MN-major operand)
//   warps 4..7   codes to bf16: each takes 32 keys of the unit, copies their codes
//                and scales two units ahead (cp.async into a ring of its own) and
//                writes code * scale, exact in bf16, into the swizzled K and V
//                rings.  Against a bf16 cache this is what the kernel adds: about
//                320 instructions per thread and unit beside the softmax's 2000
//                issue slots.
//   warps 8..15  softmax: one thread per row, a quarter of a row of S at a time;
//                they also bring the next segment's queries (cp.async)
// A key that a row does not see must not reach it.  Its S is replaced by -inf;
// its value has the probability 0, and 0 times a value must be 0: slots past a
// sequence's length are written as zeros, and a value group whose scale is NaN
// (an input's NaN or infinity) is written as zeros and flagged, and the rows
// that see it are made NaN at the end.
#pragma once
#include "attention_tc.cuh"
#include "kv_attention.cuh"

namespace vla {
namespace kv {
namespace tc {

constexpr int BQ = 128;
constexpr int kRows = 2 * BQ;  // room for rows of an item (it has the whole query tokens that fit)
constexpr int kKeys = 128;     // keys of a unit
constexpr int kThreads = 512;
constexpr int kLaunchRegs = 128;  // 65536 / 512
constexpr int kIssueRegs = 88;    // warps 0..3
constexpr int kCodeRegs = 88;     // warps 4..7
constexpr int kSoftRegs = 168;    // warps 8..15
static_assert(kIssueRegs + kCodeRegs + 2 * kSoftRegs == 4 * kLaunchRegs, "register split must equal the launch total");
constexpr int kRing = 3;    // K and V tiles
constexpr int kFlags = 4;   // flag sets: a softmax thread reads set j before S(j+1) may be issued
constexpr int TILE_BYTES = kKeys * HD * 2;
constexpr uint32_t S_COL0 = 0, P_COL0 = 256, O_COL0 = 384;
constexpr float kRescaleLog2 = 8.f;

// What a converting warp copies: half a page.
template <int BITS>
struct Raw {
  static constexpr int kCodes = kUnit / 2 * HD * BITS / 8;  // bytes of 32 keys' (or values') codes
  static constexpr int kBytes = 2 * kCodes + 256;
  static constexpr int kStages = 3;
};

struct Flags {
  uint32_t nan[2][4];  // per value group: keys whose scale is NaN
  uint32_t absent[4];  // per 32 keys: not there
};

// A CTA's share of an item, as warp 0 hands it to the other roles.
struct Segment {
  Span sp;
  int b, h, r0;        // sequence, kv head, first row
  int u0, n;           // units [u0, u0 + n)
  int whole;           // ... are all of the item's
  int more;            // another segment follows
  long long slot;      // of its part in the workspace, in rows
};
// Entries: one is written again when both softmax groups have seen its last P.V done.
constexpr int kSegments = 8;

template <int BITS>
struct Smem {
  uint8_t q[2][2][TILE_BYTES];  // [buffer][tile]
  uint8_t k[kRing][TILE_BYTES];
  uint8_t v[kRing][TILE_BYTES];
  uint8_t raw[4][Raw<BITS>::kStages][Raw<BITS>::kBytes];  // [warp]
  Flags flags[kFlags];
  Segment seg[kSegments];
  uint64_t seg_full[kSegments], seg_empty[kSegments];
  uint64_t q_full[2][2];  // [buffer][group]
  uint64_t k_full[kRing], k_empty[kRing];
  uint64_t v_full[kRing], v_empty[kRing];
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];
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

// 32 keys' codes to rows [r0, r0 + 32) of a K and a V tile.
template <int BITS>
__device__ __forceinline__ void convert(uint32_t raw, uint32_t kt, uint32_t vt, int r0, int live, bool clean,
                                        uint32_t mask, int lane) {
  constexpr int C = Raw<BITS>::kCodes;
  const int g = lane >> 2, t = lane & 3;
#pragma unroll 1
  for (int tile = 0; tile < 2; ++tile) {
    const uint32_t sc = raw + 2 * C + tile * 128;
    // keys: tokens a and a + 2, 8 dims of either group
    const int a = 4 * (g >> 1) + (g & 1);
    uint4 d = lds16(sc + g * 16);
    const int row = r0 + tile * 16 + a;
#pragma unroll
    for (int n = 0; n < 2; ++n) {  // odd g the other way round: eight lanes then touch all banks
      const int grp = n ^ (g & 1);
      uint32_t c[2][4];
      if (BITS == 4) {
        const uint4 w = lds16(raw + tile * 512 + lane * 16);
        codes4(grp == 0 ? w.x : w.y, mask, c[0]);
        codes4(grp == 0 ? w.z : w.w, mask, c[1]);
      } else {
        const uint4 w = lds16(raw + tile * 1024 + grp * 512 + lane * 16);
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
      w0 = lds16(raw + C + tile * 512 + lane * 16);
    } else {
      w0 = lds16(raw + C + tile * 1024 + lane * 16);
      w1 = lds16(raw + C + tile * 1024 + 512 + lane * 16);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int rr = r0 + tile * 16 + 4 * q + r;
      uint32_t d0 = lo2(vs[r]), d1 = hi2(vs[r]);
      if (!clean) {  // past the end, or NaN (flagged)
        const bool past = 4 * q + r + tile * 16 >= live;
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

// A finished row of O_g: divided by its sum to the output, or as it is to the
// CTA's part slot.  The caller has waited for the last P.V.
__device__ __forceinline__ void finish_row(const AttnParams& p, uint32_t o_adr, float m, float l, uint32_t nan, int b,
                                           int h, int ql, int row, bool there, bool whole, long long slot) {
  const int i = row / p.G, head = h * p.G + row - i * p.G;
  const bool empty = i >= ql || l == 0.f;
  const float inv = !whole ? 1.f : empty ? 0.f : 1.f / l;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    float o[HD / 2];
    tmem_ld32(o_adr + (uint32_t)half * (HD / 2), o);  // warp-collective: every lane loads
    if ((nan >> half) & 1u) {
#pragma unroll
      for (int c = 0; c < HD / 2; ++c) o[c] = __uint_as_float(0x7FC00000u);
    }
    if (there) {
      if (whole) {
        uint4* dst = reinterpret_cast<uint4*>(p.o + (long long)b * p.o_batch + (long long)i * p.o_row +
                                              (long long)head * HD + half * (HD / 2));
#pragma unroll
        for (int c8 = 0; c8 < HD / 16; ++c8) {
          float tv8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) tv8[e] = empty && !((nan >> half) & 1u) ? 0.f : o[c8 * 8 + e] * inv;
          dst[c8] = pack_bf16x8(tv8);
        }
      } else {
        float4* dst = reinterpret_cast<float4*>(p.part_o + slot * HD + half * (HD / 2));
#pragma unroll
        for (int c4 = 0; c4 < HD / 8; ++c4)
          dst[c4] = make_float4(o[4 * c4], o[4 * c4 + 1], o[4 * c4 + 2], o[4 * c4 + 3]);
      }
    }
  }
  if (!whole && there) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m, l);
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
      mbar_init(&sm.q_full[i][0], 4);
      mbar_init(&sm.q_full[i][1], 4);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.s_free[i], 128);
      mbar_init(&sm.p_full[i], 128);
      mbar_init(&sm.pv_done[i], 1);
    }
    for (int s = 0; s < kSegments; ++s) {
      mbar_init(&sm.seg_full[s], 1);
      mbar_init(&sm.seg_empty[s], 2);
    }
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&sm.k_full[s], 4);
      mbar_init(&sm.k_empty[s], 2);
      mbar_init(&sm.v_full[s], 4);
      mbar_init(&sm.v_empty[s], 2);
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

  // this CTA's share of the units
  int left;
  Deal d;
  {
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
    __syncthreads();
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
        int group = sm.group, units = units_of(p, group), h = sm.left / units, u0 = sm.left - h * units;
#pragma unroll 1
        for (; ok && left > 0; ++it) {
          const int b = group / p.row_blocks, r0 = (group - b * p.row_blocks) * p.block;
          const int n = min(units - u0, left);
          left -= n;
          if (it >= kSegments)
            ok = mbar_wait_bounded(&sm.seg_empty[it % kSegments], ((it / kSegments) & 1) ^ 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) {
            Segment& sg = sm.seg[it % kSegments];
            sg.sp = span_of(p, b, r0, p.block);
            sg.b = b;
            sg.h = h;
            sg.r0 = r0;
            sg.u0 = u0;
            sg.n = n;
            sg.whole = n == units;
            sg.more = left > 0;
            sg.slot = (2ll * blockIdx.x + (it > 0 ? 1 : 0)) * kRows;
            mbar_arrive(&sm.seg_full[it % kSegments]);
            record_cut(p, d, group, h, u0, u0 + n, units, it);
          }
          // the next item that has units
          u0 = 0;
          if (++h == heads && left > 0) {
            h = 0;
#pragma unroll 1
            do units = units_of(p, ++group);
            while (units == 0);
          }
        }
      } else if (warp < 3) {
        // ---------------- S issuers ----------------
        const int g = warp - 1;
        constexpr uint32_t idesc_s = make_idesc_bf16(BQ, kKeys);
        const uint32_t s_tmem = tmem + S_COL0 + (uint32_t)g * kKeys;
        int t = 0;
#pragma unroll 1
        for (bool more = true; more && ok; ++it) {
          const Segment& sg = segment(it);
          if (!ok) break;
          const int n = sg.n, qb = it & 1;
          more = sg.more;
          ok = mbar_wait_bounded(&sm.q_full[qb][g], (it >> 1) & 1, abort_flag);
          const uint64_t qdesc = make_sw128_desc(smem_u32(sm.q[qb][g]));
#pragma unroll 1
          for (int j = 0; ok && j < n; ++j, ++t) {
            const int sk = t % kRing;
            ok = mbar_wait_bounded(&sm.k_full[sk], (t / kRing) & 1, abort_flag);
            if (ok && t > 0) ok = mbar_wait_bounded(&sm.s_free[g], (uint32_t)(t - 1) & 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t kdesc = make_sw128_desc(smem_u32(sm.k[sk]));
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) tc_mma_bf16(s_tmem, qdesc + 2 * k, kdesc + 2 * k, idesc_s, k > 0);
              tc_commit(&sm.s_full[g]);
              tc_commit(&sm.k_empty[sk]);
            }
            __syncwarp();
          }
        }
      } else {
        // ---------------- P.V issuer ----------------
        constexpr uint32_t idesc_pv = make_idesc_bf16(BQ, HD) | (1u << 16);  // B (V) is MN-major
        int t = 0;
#pragma unroll 1
        for (bool more = true; more && ok; ++it) {
          const Segment& sg = segment(it);
          if (!ok) break;
          const int n = sg.n;
          more = sg.more;
#pragma unroll 1
          for (int j = 0; ok && j < n; ++j, ++t) {
            const int sv = t % kRing;
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
              ok = mbar_wait_bounded(&sm.p_full[g], (uint32_t)t & 1u, abort_flag);
              if (ok) ok = mbar_wait_bounded(&sm.v_full[sv], (t / kRing) & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) {
                const uint32_t p_tmem = tmem + P_COL0 + (uint32_t)g * (kKeys / 2);
                const uint32_t o_tmem = tmem + O_COL0 + (uint32_t)g * HD;
                const uint32_t vbase = smem_u32(sm.v[sv]);
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                  attn_tc::tc_mma_bf16_ts(o_tmem, p_tmem + (uint32_t)k * 8u,
                                          attn_tc::make_sw128_mn_desc(vbase + (uint32_t)k * 2048u, 16384u), idesc_pv,
                                          (j > 0 || k > 0) ? 1u : 0u);
                tc_commit(&sm.pv_done[g]);
                tc_commit(&sm.v_empty[sv]);
              }
              __syncwarp();
            }
          }
        }
      }
    } else if (warp < 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCodeRegs));
      // ---------------- codes to bf16 ----------------
      using Rw = Raw<BITS>;
      const int w = warp - 4;  // keys [32 w, 32 w + 32) of a unit: half (w & 1) of page w >> 1
      const uint32_t raw = smem_u32(sm.raw[w]);
      // copies run kStages - 1 units ahead, with a segment count of their own
      int ci = 0, cu = 0, cn = 0, ct = 0, cpage = 0, cb = 0, ch = 0;
      int csink = 0, cfirst = 0, ccount = 0;
      bool cmore = true;
      uint32_t there = 0;  // bit (stage): the page exists
      auto page_ahead = [&]() {  // the next copy's page number
        const int u = 2 * cu + (w >> 1);
        if (u < ccount) cpage = p.c.table[(long long)cb * p.c.table_ld + (u < csink ? u : cfirst + u - csink)];
      };
      auto copy_segment = [&]() {
        const Segment& sg = segment(ci);
        ++ci;
        if (!ok) return;
        cu = sg.u0;
        cn = sg.n;
        cb = sg.b;
        ch = sg.h;
        csink = sg.sp.sink;
        cfirst = sg.sp.first;
        ccount = sg.sp.count;
        cmore = sg.more;
        page_ahead();
      };
      copy_segment();
      auto copy_next = [&]() {
        if (cn == 0 && cmore) copy_segment();
        if (cn > 0 && ok) {
          const int st = ct % Rw::kStages, u = 2 * cu + (w >> 1);
          bool have = false;
          if (u < ccount) {
            have = cpage >= 0 && cpage < p.c.pages;
            if (have) {
              const uint8_t* blk = p.c.pool + ((long long)cpage * heads + ch) * Block<BITS>::kBytes;
              const uint32_t dst = raw + st * Rw::kBytes + lane * 16;
              const uint8_t* src = blk + (w & 1) * Rw::kCodes + lane * 16;
#pragma unroll
              for (int i = 0; i < Rw::kCodes / 512; ++i) {
                copy16(dst + i * 512, src + i * 512);
                copy16(dst + Rw::kCodes + i * 512, src + Block<BITS>::kValues + i * 512);
              }
              if (lane < 16)
                copy16(dst + 2 * Rw::kCodes, blk + Block<BITS>::kScales + (w & 1) * 256 + lane * 16);
            } else {
              vla_record_error(VLA_DERR_KV_RANGE);
            }
          }
          there = have ? there | (1u << st) : there & ~(1u << st);
          ++ct;
          ++cu;
          if (--cn > 0)
            page_ahead();
          else if (cmore && __all_sync(0xffffffffu, mbar_test(&sm.seg_full[ci % kSegments], (ci / kSegments) & 1)))
            copy_segment();
        }
        copy_commit();
      };
#pragma unroll
      for (int i = 0; i < Rw::kStages - 1; ++i) copy_next();
      int t = 0;
#pragma unroll 1
      for (bool more = ok; more && ok; ++it) {
        const Segment& sg = segment(it);
        if (!ok) break;
        const int n = sg.n, u0 = sg.u0, len = sg.sp.len, sink = sg.sp.sink, first = sg.sp.first;
        more = sg.more;
#pragma unroll 1
        for (int j = 0; ok && j < n; ++j, ++t) {
          const int st = t % Rw::kStages, sr = t % kRing;
          const bool have = (there >> st) & 1u;  // before copy_next changes another stage's bit
          copy_next();
          copy_wait<Rw::kStages - 1>();
          __syncwarp();
          ok = mbar_wait_bounded(&sm.k_empty[sr], ((t / kRing) & 1) ^ 1, abort_flag);
          if (ok) ok = mbar_wait_bounded(&sm.v_empty[sr], ((t / kRing) & 1) ^ 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t kt = smem_u32(sm.k[sr]), vt = smem_u32(sm.v[sr]), from = raw + st * Rw::kBytes;
          const int u = 2 * (u0 + j) + (w >> 1), page = u < sink ? u : first + u - sink;
          int live = 0;  // of the 32 keys, those inside the sequence
          uint32_t n0 = 0u, n1 = 0u;
          if (have) {
            live = min(32, len - (page * kUnit + (w & 1) * 32));
            // key `lane`: tile lane / 16, token 4 q + b + 2 c at (2 q + b) * 16 + c * 8
            const int tk = lane & 15;
            uint32_t s;
            asm volatile("ld.shared.u32 %0, [%1];"
                         : "=r"(s)
                         : "r"(from + 2 * Rw::kCodes + (lane >> 4) * 128 + (2 * (tk >> 2) + (tk & 1)) * 16 +
                               ((tk >> 1) & 1) * 8 + 4));
            n0 = __ballot_sync(0xffffffffu, lane < live && (s & 0x7F80u) == 0x7F80u);
            n1 = __ballot_sync(0xffffffffu, lane < live && (s & 0x7F800000u) == 0x7F800000u);
            convert<BITS>(from, kt, vt, w * 32, live, live == 32 && (n0 | n1) == 0u, p.mask, lane);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              sts16(kt + w * 4096 + i * 512 + lane * 16, 0u, 0u, 0u, 0u);
              sts16(vt + w * 4096 + i * 512 + lane * 16, 0u, 0u, 0u, 0u);
            }
          }
          if (lane == 0) {
            Flags& f = sm.flags[t % kFlags];
            f.nan[0][w] = n0;
            f.nan[1][w] = n1;
            f.absent[w] = have ? 0u : 1u;
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sm.k_full[sr]);
            mbar_arrive(&sm.v_full[sr]);
          }
        }
      }
      copy_wait<0>();
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
      // ---------------- softmax / output ----------------
      const int g = (warp - 8) >> 2, q = warp & 3;
      const uint32_t lane_base = (uint32_t)(q * 32) << 16;
      const uint32_t s_adr = tmem + lane_base + S_COL0 + (uint32_t)g * kKeys;
      const uint32_t p_adr = tmem + lane_base + P_COL0 + (uint32_t)g * (kKeys / 2);
      const uint32_t o_adr = tmem + lane_base + O_COL0 + (uint32_t)g * HD;
      int t = 0;
      // a segment's O_g is read out before the next one's first P_g is released, so that
      // its last P.V runs beside the next one's S
      bool pending = false, pend_there = false, pend_whole = false;
      int pend_b = 0, pend_h = 0, pend_ql = 0, pend_row = 0;
      long long pend_slot = 0;
      float pend_m = 0.f, pend_l = 0.f;
      uint32_t pend_nan = 0;
      // segment i's queries to their buffer: each warp its 32 rows, 4 rows an instruction
      auto fetch_q = [&](int i) {
        const Segment& sg = segment(i);
        if (!ok) return;
        const uint32_t dst = smem_u32(sm.q[i & 1][g]) + q * 4096;
        const bf16* src = p.q + (long long)sg.b * p.q_batch + (long long)sg.h * p.G * HD + (lane & 7) * 8;
        int row = sg.r0 + g * BQ + q * 32 + (lane >> 3), qi = row / p.G, hh = row - qi * p.G;
        const int di = 4 / p.G, dh = 4 - di * p.G;
#pragma unroll 1
        for (int r = lane >> 3; r < 32; r += 4, row += 4) {
          const bool there = row < rows;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           dst + r * 128 + (((lane & 7) ^ (r & 7)) << 4)),
                       "l"(there ? src + (long long)qi * p.q_row + hh * HD : p.q), "r"(there ? 16 : 0)
                       : "memory");
          qi += di;
          hh += dh;
          if (hh >= p.G) {
            hh -= p.G;
            ++qi;
          }
        }
        copy_commit();
      };
      auto post_q = [&](int i) {
        copy_wait<0>();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[i & 1][g]);
      };
      fetch_q(0);
      post_q(0);
#pragma unroll 1
      for (bool more = true; ok; ++it) {
        if (!more) break;
        const Segment& sg = segment(it);
        if (!ok) break;
        more = sg.more;
        // (the buffer's last reader, S of the segment before, is done)
        if (more) fetch_q(it + 1);
        if (!ok) break;
        const Span sp = sg.sp;
        const int u0 = sg.u0, n = sg.n, r0 = sg.r0;
        const int row = r0 + g * BQ + q * 32 + lane, i = row / p.G;
        const bool mine = row < rows && row < r0 + p.block;
        const int pos = mine && i < sp.ql ? sp.pos(i, p.causal) : -1;
        const bool idle = r0 + g * BQ + q * 32 >= rows;  // no row in this warp
        float m = -INFINITY, l = 0.f;
        uint32_t nan = 0;
#pragma unroll 1
        for (int j = 0; j < n; ++j, ++t) {
          ok = mbar_wait_bounded(&sm.s_full[g], (uint32_t)t & 1u, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int ua = 2 * (u0 + j), ka = sp.unit(ua), kb = sp.unit(ua + 1);  // pages
          bool plain = ((ka >= sp.open && ka < sp.shut) || ka < sp.sink_open) &&
                       ((kb >= sp.open && kb < sp.shut) || kb < sp.sink_open);
          uint32_t vis[4] = {0u, 0u, 0u, 0u};  // keys that the row sees, set where not all are
          {
            const uint32_t f = smem_u32(&sm.flags[t % kFlags]);
            const uint4 n0 = lds16(f), n1 = lds16(f + 16), ab = lds16(f + 32);
            const uint32_t flagged = n0.x | n0.y | n0.z | n0.w | n1.x | n1.y | n1.z | n1.w;
            plain = plain && (ab.x | ab.z) == 0u;
            if (!plain || flagged != 0u) {
              vis[0] = ab.x != 0u ? 0u : seen32(ka * kUnit, pos, p.window, p.sinks);
              vis[1] = ab.x != 0u ? 0u : seen32(ka * kUnit + 32, pos, p.window, p.sinks);
              vis[2] = ab.z != 0u ? 0u : seen32(kb * kUnit, pos, p.window, p.sinks);
              vis[3] = ab.z != 0u ? 0u : seen32(kb * kUnit + 32, pos, p.window, p.sinks);
              if (((n0.x & vis[0]) | (n0.y & vis[1]) | (n0.z & vis[2]) | (n0.w & vis[3])) != 0u) nan |= 1u;
              if (((n1.x & vis[0]) | (n1.y & vis[1]) | (n1.z & vis[2]) | (n1.w & vis[3])) != 0u) nan |= 2u;
            }
          }
          // The row goes by in quarters, the next one on its way from TMEM.  Exponentials
          // are taken against the maximum so far while the unit's own is still being
          // found; where that outgrows it by more than 2^8 (the first unit, then rarely)
          // the quarters are gone through again.
          uint32_t sa[2][32];
          auto mask = [&](uint32_t* r, int qt) {
            if (!plain) {
              const uint32_t v = qt == 0 ? vis[0] : qt == 1 ? vis[1] : qt == 2 ? vis[2] : vis[3];
#pragma unroll
              for (int c = 0; c < 32; ++c) r[c] = (v >> c) & 1u ? r[c] : 0xFF800000u;
            }
          };
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          auto top = [&](const uint32_t* r) {
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) mx4[e] = max3(mx4[e], __uint_as_float(r[c + e]), __uint_as_float(r[c + 4 + e]));
            }
          };
          float rs[4] = {0.f, 0.f, 0.f, 0.f};
          auto exps = [&](const uint32_t* r, int qt) {
            const float mbase = m == -INFINITY ? 0.f : m;
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float x0, x1, e0, e1;
              attn_tc::fma2(__uint_as_float(r[c]), __uint_as_float(r[c + 1]), p.scale_log2, -mbase, x0, x1);
              e0 = ex2(x0);
              e1 = ex2(x1);
              attn_tc::add2(rs[c & 2], rs[(c & 2) + 1], e0, e1);
              pk[c >> 1] = pack_bf16x2(e0, e1);
            }
            tmem_put16(p_adr + qt * 16, pk);
          };
          if (!idle) tmem_start32(s_adr, sa[0]);
          if (t > 0) {
            // P_g and O_g were last used by P.V of unit t - 1
            ok = mbar_wait_bounded(&sm.pv_done[g], (uint32_t)(t - 1) & 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
          }
          if (j == 0 && pending) {
            if (q == 0 && lane == 0) mbar_arrive(&sm.seg_empty[(it - 1) % kSegments]);
            finish_row(p, o_adr, pend_m, pend_l, pend_nan, pend_b, pend_h, pend_ql, pend_row, pend_there, pend_whole, pend_slot);
          }
          if (!idle) {
            if (j == 0) {  // no maximum yet: the unit's own, first
#pragma unroll 1
              for (int qt = 0; qt < 4; qt += 2) {
                tmem_wait32(sa[0]);
                tmem_start32(s_adr + 32 * qt + 32, sa[1]);
                mask(sa[0], qt);
                top(sa[0]);
                tmem_wait32(sa[1]);
                tmem_start32(s_adr + (qt == 0 ? 64 : 0), sa[0]);
                mask(sa[1], qt + 1);
                top(sa[1]);
              }
              m = max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3])) * p.scale_log2;
            }
            bool again = false;
            float mx = m;
#pragma unroll 1
            for (int qt = 0; qt < 4; qt += 2) {
              tmem_wait32(sa[0]);
              tmem_start32(s_adr + 32 * qt + 32, sa[1]);
              mask(sa[0], qt);
              top(sa[0]);
              exps(sa[0], qt);
              tmem_wait32(sa[1]);
              if (qt == 0) tmem_start32(s_adr + 64, sa[0]);
              mask(sa[1], qt + 1);
              top(sa[1]);
              if (qt == 2) {
                mx = max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3])) * p.scale_log2;
                again = __any_sync(0xffffffffu, mx > m + kRescaleLog2);
                if (!again) {
                  tc_fence_before();
                  mbar_arrive(&sm.s_free[g]);
                }
              }
              exps(sa[1], qt + 1);
            }
            if (again) {
              float alpha = 1.f;
              if (mx > m + kRescaleLog2) {
                alpha = ex2(m - mx);
                m = mx;
                l *= alpha;
              }
#pragma unroll 1
              for (int c = 0; c < HD; c += 16) {
                float o[16];
                uint32_t u[16];
                tmem_ld16(o_adr + c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * alpha);
                attn_tc::tmem_st16(o_adr + c, u);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) rs[e] = 0.f;
              tmem_put_wait();
#pragma unroll 1
              for (int qt = 0; qt < 4; ++qt) {
                tmem_start32(s_adr + 32 * qt, sa[0]);
                tmem_wait32(sa[0]);
                if (qt == 3) {
                  tc_fence_before();
                  mbar_arrive(&sm.s_free[g]);
                }
                mask(sa[0], qt);
                exps(sa[0], qt);
              }
            }
            tmem_put_wait();
            const float sum = (rs[0] + rs[1]) + (rs[2] + rs[3]);
            l += sum;
          } else {
            tc_fence_before();
            mbar_arrive(&sm.s_free[g]);
          }
          tc_fence_before();
          mbar_arrive(&sm.p_full[g]);
        }
        if (!ok) break;
        if (more) post_q(it + 1);
        pending = true;
        pend_whole = sg.whole != 0;
        pend_b = sg.b, pend_h = sg.h, pend_ql = sp.ql, pend_row = row, pend_there = mine, pend_m = m, pend_l = l, pend_nan = nan;
        pend_slot = sg.slot + (row - r0);
      }
      if (ok && pending) {
        ok = mbar_wait_bounded(&sm.pv_done[g], (uint32_t)(t - 1) & 1u, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          tc_fence_after();
          finish_row(p, o_adr, pend_m, pend_l, pend_nan, pend_b, pend_h, pend_ql, pend_row, pend_there, pend_whole, pend_slot);
        }
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
