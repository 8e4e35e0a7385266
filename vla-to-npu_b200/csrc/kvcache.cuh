// Quantised key/value cache, head_dim 64: the block layout, the kernel that
// quantises rows as it writes them and the one that reads them back.
//
// A cache is a pool of pages of 64 tokens; a page holds one block per kv head.
// Block: key codes | value codes | scales (4 bits: 2048 + 2048 + 512 bytes,
// 8 bits: 4096 + 4096 + 512 bytes), tokens in tiles of 16.
//
// Quantisation of a group of 32 elements (two groups per row of 64), a = max |x|:
//   4 bits: d = a / 8 with its magnitude rounded UP to 5 significant bits, so
//           that |x / d| <= 8; d is negative when the largest magnitude is a
//           positive element only, so that it takes code -8 (the code range
//           [-8, 7] has one more negative code);
//           code = min(rint(x / d), 7), stored plus 8.
//   8 bits: d = the smallest power of two with 127 d >= a; code = rint(x / d).
// d >= 2^-100; d = NaN when a is not below 2^127 (NaN and infinities included).
// A 4-bit code has at most 3 significant bits and a 4-bit d five, an 8-bit
// code at most 7 and an 8-bit d one, so code * d is a bf16 number EXACTLY: the
// cache stands for bf16 keys and values, and every reader (this file's, and the
// attention kernels' products with the scales applied before or after) sees the
// same numbers without another rounding.
//
// Order inside a tile.  The attention kernel feeds keys and values to
// mma.m16n8k16 as the 16-row operand, straight from global memory to registers:
// lane (g = lane / 4, t = lane % 4) needs for its key rows g and g + 8 the same
// 16 dims, and for its value columns 2t, 2t+1, 2t+8, 2t+9 (tokens) the same 8
// dims.  Rows are taken as tokens 4(g/2) + g%2 and that + 2, columns as tokens
// 4t .. 4t+3, which makes both a 16-byte load per lane, contiguous over the warp:
//   keys   4 bits: 16 bytes at (2q + b) * 64 + t * 16 = [token 4q+b: word of
//          dims 8t.. of group 0, of group 1; token 4q+b+2: the same]
//   values 4 bits: 16 bytes at q * 128 + g * 16 = [word of token 4q + r: dims
//          4g..4g+3 of group 0, then of group 1; r = 0..3]
//   8 bits: the same with a 512-byte half tile per group: keys [token 4q+b: 8
//          bytes; token 4q+b+2: 8 bytes], values [4 bytes of token 4q + r]
//   scales: 8 bytes per token [key d0, d1, value d0, d1] at (2q + b) * 16 + c * 8
//          for token 4q + b + 2c.
// A 4-bit word holds element 2i in bits 4i and element 2i+1 in bits 16 + 4i; an
// 8-bit word of 4 has the byte order 0, 2, 1, 3: masking (and shifting) a word
// then gives pairs of neighbours in its two halves.
#pragma once
#include "common.cuh"

namespace vla {
namespace kv {

constexpr int kPage = 64;  // tokens per page
constexpr int HD = 64;
constexpr int kTile = 16;

template <int BITS>
struct Block {
  static constexpr int kTileCodes = kTile * HD * BITS / 8;      // bytes of a tile's key (or value) codes
  static constexpr int kValues = kPage * HD * BITS / 8;         // offset of the value codes
  static constexpr int kScales = 2 * kValues;                   // offset of the scales
  static constexpr int kBytes = kScales + kPage * 8;            // 4608 or 8704
};

struct Cache {
  uint8_t* pool;
  const int* table;
  long long table_ld;
  int pages, max_pages, batch, kv_heads;
};

// Block of (sequence b, page slot, kv head); null, with the error recorded,
// when the slot or the page number is out of range.
template <int BITS>
__device__ __forceinline__ uint8_t* block_of(const Cache& c, int b, int slot, int h) {
  if (slot < 0 || slot >= c.max_pages) {
    vla_record_range();
    return nullptr;
  }
  const int page = c.table[(long long)b * c.table_ld + slot];
  if (page < 0 || page >= c.pages) {
    vla_record_range();
    return nullptr;
  }
  return c.pool + ((long long)page * c.kv_heads + h) * Block<BITS>::kBytes;
}

// ---------------------------------------------------------------------------
// word <-> numbers
// ---------------------------------------------------------------------------
__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t*>(&h); }

// (a & mask) | bits in one instruction.  It takes one immediate only, so a mask
// that is a constant to the compiler costs a second one: the attention kernel
// passes it as a launch argument.
__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}

// mask selects a code's magnitude bits in both halves: the low ones of a code.
template <int BITS>
constexpr uint32_t code_mask() {
  return BITS == 4 ? 0x000F000Fu : 0x007F007Fu;
}

// The codes of a 4-bit word as bf16 pairs: 128 + n sits in the mantissa of
// 0x4300 | n; subtracting 136 = 128 + 8 is exact.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t mask, uint32_t* p) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = as_u32(__hsub2(as_bf2(lop_and_or(w >> (4 * i), mask, 0x43004300u)), as_bf2(0x43084308u)));
}

// The codes of an 8-bit word (two's complement bytes) as two bf16 pairs: 128 +
// the low seven bits, minus 128 or 256 by the sign bit (0x4380 is 256); exact.
__device__ __forceinline__ void codes8(uint32_t w, uint32_t mask, uint32_t* p) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = w >> (8 * i);
    p[i] = as_u32(__hsub2(as_bf2(lop_and_or(u, mask, 0x43004300u)), as_bf2(lop_and_or(u, mask + 0x00010001u, 0x43004300u))));
  }
}

// Scale of a group from its largest positive and largest negative magnitude
// (bf16 bits; below 0 where no element has that sign, but the larger one >= 0).
template <int BITS>
__device__ __forceinline__ float group_scale(int hp, int hn) {
  const int top = max(hp, hn);
  const float a = __uint_as_float((uint32_t)top << 16);
  float d;
  if (BITS == 4) {
    // a / 8 up to 5 significant bits: 4 of the 23 mantissa bits stay
    d = __uint_as_float((__float_as_uint(a * 0.125f) + 0x0007FFFFu) & ~0x0007FFFFu);
    d = fmaxf(d, 0x1p-100f);
    if (hp > max(hn, 0)) d = -d;
  } else {
    // a in [2^k, 2^(k+1)): 127 * 2^(k-6) reaches it or 127 * 2^(k-5) does
    const float p = __uint_as_float(__float_as_uint(a) & 0x7F800000u) * 0x1p-6f;
    d = fmaxf(127.f * p >= a ? p : 2.f * p, 0x1p-100f);
  }
  return top >= 0x7F00 ? __uint_as_float(0x7FC00000u) : d;  // 0x7F00 is 2^127
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes of 8 elements with the scale's reciprocal r.
// 4 bits: x r differs from x / d by less than 2^-20 (r is the hardware's reciprocal, off by
// an ulp at most), while a quotient of an
// 8-bit by a 5-bit significand that is no tie lies at least 2^-11 from every
// half-integer within [-8.5, 8.5] (its distance is a multiple of 2^-5 / 62 when
// it is near one at all).  The fused multiply-add onto 1.5 * 2^12 rounds to
// multiples of 2^-11, which makes ties exact again and moves nothing else
// across one; the addition of 1.5 * 2^23 rounds to integers, ties to even.  The
// codes + 8 stay floats until a half-word is summed (base 16, below 2^16: exact), two
// half-words per instruction, which spares the integer pipe the shifts.
__device__ __forceinline__ uint32_t pack4(const float* x, float r) {
  auto both = [](float v) { return make_float2(v, v); };
  float2 w = both(0.f);
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    float2 q = __fadd2_rn(__ffma2_rn(make_float2(x[2 * i], x[2 * i + 1]), both(r), both(6144.f)), both(-6144.f));
    q.x = fminf(q.x, 7.f);
    q.y = fminf(q.y, 7.f);
    q = __fadd2_rn(__fadd2_rn(q, both(12582912.f)), both(-12582904.f));
    w = i == 3 ? q : __ffma2_rn(w, both(16.f), q);
  }
  w = __fadd2_rn(w, both(8388608.f));  // 2^23: the sum in the low mantissa bits
  return __byte_perm(__float_as_uint(w.x), __float_as_uint(w.y), 0x5410);
}
// 8 bits: d is a power of two, so x r is exact and one rounding does it.
__device__ __forceinline__ uint32_t pack8(const float* x, float r) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t n = __float_as_uint(fmaf(x[e], r, 12582912.f)) & 255u;
    w |= n << (16 * (e & 1) + 8 * (e >> 1));
  }
  return w;
}

// The largest positive and negative magnitudes of 8 bf16 (bits, as signed 16-bit
// halves [positive | negative]) over the 4 lanes of a group.
__device__ __forceinline__ uint32_t group_top(const uint4& u) {
  const uint32_t f = 0x80008000u;
  uint32_t hp = __vmaxs2(__vmaxs2(u.x, u.y), __vmaxs2(u.z, u.w));
  uint32_t hn = __vmaxs2(__vmaxs2(u.x ^ f, u.y ^ f), __vmaxs2(u.z ^ f, u.w ^ f));
  uint32_t m = __vmaxs2(__byte_perm(hp, hn, 0x5410), __byte_perm(hp, hn, 0x7632));  // low half: positive
  m = __vmaxs2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return __vmaxs2(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

// Loads that keep nothing in L1: the cache and the rows are read once, and with
// launch overlap an earlier kernel's line must not outlive the write between.
__device__ __forceinline__ uint32_t ld_stream1(const void* p) {
  uint32_t v;
  asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream2(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendParams {
  Cache c;
  const bf16* k;
  const bf16* v;
  long long k_row, v_row, k_batch, v_batch;
  const int* start;
  const int* count;  // valid tokens per sequence, or null
  int n;             // tokens per sequence
  int quads;         // aligned groups of 4 positions that n tokens can touch
};

// One warp takes QUADS neighbouring groups of 4 aligned cache positions of a
// (sequence, kv head), lane = (token r, 8 dims w) of each.  blockIdx.x: (groups,
// kv head), blockIdx.y: sequence.  Four groups keep four times the loads in flight
// and share the coordinates' arithmetic, one is a shorter chain: reading 32
// histories of up to 8001 tokens 64.5 us with four, 77.0 with one; a single
// sequence's 113 tokens 2.8 and 1.7 us.  kv_host.cuh takes four where that still
// fills the SMs' 64 warps.

struct Lane {
  int token, slot, off;  // index of the lane's token among the n, page slot, position in the page
  bool live;
};
__device__ __forceinline__ Lane lane_of(int start, int valid, int quad, int lane) {
  Lane it;
  const uint32_t pos = (((uint32_t)start >> 2) + (uint32_t)quad) * 4u + (uint32_t)(lane >> 3);  // below 2^32
  it.token = (int)(pos - (uint32_t)start);
  it.slot = (int)(pos / kPage);
  it.off = (int)(pos % kPage);
  it.live = start >= 0 && it.token >= 0 && it.token < valid;
  return it;
}

// Each lane loads 16 bytes of K and of V per group (a token's 128-byte row by 8
// lanes), takes the scale over the 4 lanes of a group of dims, and the warp
// writes whole 128-byte lines of codes (the order inside a tile keeps a group's
// words together).  Bound by its instructions at this size: 256 sequences of 113
// rows (15 / 5 heads, 4 bits), written and read back, take 26.5 us of which the bytes
// need 15; 16 x 4001 rows in 8 bits 48 of 39 us.  Four CTAs per SM cost it 3 spilled
// registers at most and gain a resident CTA: three 27.2 and 50.0 us, five (more
// spills) 27.3 and 50.6.  Reading alone comes to 0.91 of the measured copy rate (32 x
// 8001 tokens, 65 us).
template <int BITS, int QUADS>
__global__ void __launch_bounds__(256, QUADS == 4 ? 4 : 1) append_kernel(AppendParams p) {
  pdl_prologue();
  using B = Block<BITS>;
  const int lane = threadIdx.x & 31, w = lane & 7;
  const int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int q0 = item / p.c.kv_heads * QUADS, h = item % p.c.kv_heads;
  if (q0 >= p.quads) return;
  for (int b = blockIdx.y; b < p.c.batch; b += gridDim.y) {
    const int s = p.start[b];
    const int valid = p.count != nullptr ? min(p.n, p.count[b]) : p.n;
    if (s < 0) vla_record_range();
    const bf16* kb = p.k + (long long)b * p.k_batch + h * HD + w * 8;
    const bf16* vb = p.v + (long long)b * p.v_batch + h * HD + w * 8;
    Lane it[QUADS];
    uint4 x[QUADS][2];
    uint8_t* blk[QUADS];
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      it[u] = lane_of(s, valid, q0 + u, lane);
      x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
      blk[u] = nullptr;
      if (it[u].live) {
        x[u][0] = ld_stream(kb + (long long)it[u].token * p.k_row);
        x[u][1] = ld_stream(vb + (long long)it[u].token * p.v_row);
        blk[u] = block_of<BITS>(p.c, b, it[u].slot, h);
      }
    }
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      const int tile = it[u].off >> 4, q = (it[u].off >> 2) & 3, r = it[u].off & 3, t = w & 3, grp = w >> 2;
      uint32_t dd[2];  // scales (bf16 bits)
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // K, V
        const uint32_t top = group_top(x[u][j]);
        const float d = group_scale<BITS>((int)(short)(top & 0xFFFFu), (int)(short)(top >> 16));
        dd[j] = __float_as_uint(d) >> 16;
        float f[8];
        unpack_bf16x8(x[u][j], f);
        const float inv = BITS == 4 ? rcp(d) : __uint_as_float(0x7F000000u - __float_as_uint(d));  // 2^-k of 2^k
        uint8_t* base = blk[u] + (j == 0 ? 0 : B::kValues) + tile * B::kTileCodes;
        if (BITS == 4) {
          const uint32_t word = pack4(f, inv);
          if (j == 0) {
            if (blk[u])
              *reinterpret_cast<uint32_t*>(base + (2 * q + (r & 1)) * 64 + t * 16 + (r >> 1) * 8 + grp * 4) = word;
          } else {
            // a value word joins 4 dims of each group: swap halves with the other group's lane
            const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 4);
            const uint32_t out = grp == 0 ? __byte_perm(word, other, 0x6240) : __byte_perm(other, word, 0x7351);
            if (blk[u]) *reinterpret_cast<uint32_t*>(base + q * 128 + (2 * t + grp) * 16 + r * 4) = out;
          }
        } else {
          const uint32_t w0 = pack8(f, inv), w1 = pack8(f + 4, inv);
          if (blk[u]) {
            base += grp * 512 + q * 128;
            if (j == 0) {
              *reinterpret_cast<uint2*>(base + (r & 1) * 64 + t * 16 + (r >> 1) * 8) = make_uint2(w0, w1);
            } else {
              *reinterpret_cast<uint32_t*>(base + (2 * t) * 16 + r * 4) = w0;
              *reinterpret_cast<uint32_t*>(base + (2 * t + 1) * 16 + r * 4) = w1;
            }
          }
        }
      }
      const uint32_t mine = dd[0] | dd[1] << 16;
      const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 4);
      if (blk[u] && w == 0)
        *reinterpret_cast<uint2*>(blk[u] + B::kScales + tile * 128 + (2 * q + (r & 1)) * 16 + (r >> 1) * 8) =
            make_uint2(__byte_perm(mine, other, 0x5410), __byte_perm(mine, other, 0x7632));
    }
  }
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
struct ReadParams {
  Cache c;
  bf16* k;
  bf16* v;
  long long k_row, v_row, k_batch, v_batch;
  const int* start;  // or null: 0
  const int* count;  // valid tokens from start on per sequence, or null: n
  int n, quads;
  uint32_t mask;     // code_mask<BITS>()
};

// The same mapping backwards; tokens past count are written as zeros.
template <int BITS, int QUADS>
__global__ void __launch_bounds__(256) read_kernel(ReadParams p) {
  pdl_prologue();
  using B = Block<BITS>;
  const int lane = threadIdx.x & 31, w = lane & 7, t = w & 3, grp = w >> 2;
  const int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int q0 = item / p.c.kv_heads * QUADS, h = item % p.c.kv_heads;
  if (q0 >= p.quads) return;
  for (int b = blockIdx.y; b < p.c.batch; b += gridDim.y) {
    const int s = p.start != nullptr ? p.start[b] : 0;
    const int valid = p.count != nullptr ? min(p.n, p.count[b]) : p.n;
    if (s < 0) vla_record_range();
    bf16* kd = p.k + (long long)b * p.k_batch + h * HD + w * 8;
    bf16* vd = p.v + (long long)b * p.v_batch + h * HD + w * 8;
    Lane it[QUADS];
    const uint8_t* blk[QUADS];
    uint32_t a[QUADS][2][2];
    uint2 sc[QUADS];
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      it[u] = lane_of(s, valid, q0 + u, lane);
      blk[u] = it[u].live ? block_of<BITS>(p.c, b, it[u].slot, h) : nullptr;
    }
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      const int tile = it[u].off >> 4, q = (it[u].off >> 2) & 3, r = it[u].off & 3;
      a[u][0][0] = a[u][0][1] = a[u][1][0] = a[u][1][1] = 0u;
      sc[u] = make_uint2(0u, 0u);
      if (!blk[u]) continue;
      const uint8_t* kb = blk[u] + tile * B::kTileCodes;
      const uint8_t* vb = kb + B::kValues;
      if (BITS == 4) {
        a[u][0][0] = ld_stream1(kb + (2 * q + (r & 1)) * 64 + t * 16 + (r >> 1) * 8 + grp * 4);
        a[u][1][0] = ld_stream1(vb + q * 128 + (2 * t + grp) * 16 + r * 4);
      } else {
        kb += grp * 512 + q * 128;
        vb += grp * 512 + q * 128;
        const uint2 c = ld_stream2(kb + (r & 1) * 64 + t * 16 + (r >> 1) * 8);
        a[u][0][0] = c.x;
        a[u][0][1] = c.y;
        a[u][1][0] = ld_stream1(vb + (2 * t) * 16 + r * 4);
        a[u][1][1] = ld_stream1(vb + (2 * t + 1) * 16 + r * 4);
      }
      sc[u] = ld_stream2(blk[u] + B::kScales + tile * 128 + (2 * q + (r & 1)) * 16 + (r >> 1) * 8);
    }
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      if (BITS == 4) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, a[u][1][0], 4);
        // group 0's words hold bytes 0 and 2, group 1's bytes 1 and 3 of both value words
        a[u][1][0] = grp == 0 ? __byte_perm(a[u][1][0], other, 0x6240) : __byte_perm(other, a[u][1][0], 0x7351);
      }
      if (it[u].token < 0 || it[u].token >= p.n) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t o[4] = {0u, 0u, 0u, 0u};
        if (blk[u]) {
          const uint32_t s2 = j == 0 ? sc[u].x : sc[u].y;
          const __nv_bfloat162 d = as_bf2(__byte_perm(s2, s2, grp == 0 ? 0x1010 : 0x3232));
          if (BITS == 4) {
            codes4(a[u][j][0], p.mask, o);
          } else {
            codes8(a[u][j][0], p.mask, o);
            codes8(a[u][j][1], p.mask, o + 2);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = as_u32(__hmul2(as_bf2(o[i]), d));
        }
        bf16* dst = j == 0 ? kd + (long long)it[u].token * p.k_row : vd + (long long)it[u].token * p.v_row;
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

}  // namespace kv
}  // namespace vla
