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
#pragma once
#include "kvcache.cuh"

namespace vla {
namespace kv {

constexpr int kUnit = 32;  // keys a warp takes at a time

struct AttnParams {
  Cache c;
  const bf16* q;
  bf16* o;
  long long q_row, q_batch, o_row, o_batch;
  const int* lens;   // keys of each sequence
  const int* q_len;  // valid query tokens per sequence, or null: Lq
  int Lq, Hq, G;
  int causal, window, sinks;
  float scale_log2;
  int row_blocks;    // blocks of 8 * NT rows per (sequence, kv head)
  int parts, per;    // splits along the keys: units per part
  float* part_o;     // [(b, h, row block)][part][8 NT][64], when parts > 1
  float* part_ml;    // [...][8 NT][2]
};

// What a block of rows [r0, r0 + n) of one sequence sees: units [0, sink) and
// [first, last], numbered 0 .. count - 1.
struct Span {
  int len, ql;    // keys, valid query tokens
  int lo, hi;     // positions of the first and last row's token
  int sink, first, count;
  int per;  // units of a part: the plan's, or more where the sequence is longer than the plan was made for
  __device__ __forceinline__ int unit(int u) const { return u < sink ? u : first + u - sink; }
  __device__ __forceinline__ int pos(int i, int causal) const { return causal ? len - ql + i : len - 1; }
};

__device__ __forceinline__ Span span_of(const AttnParams& p, int b, int r0, int n) {
  Span s;
  s.len = p.lens[b];
  const long long room = (long long)p.c.max_pages * kPage;
  if (s.len < 0 || s.len > room) {
    vla_record_error(VLA_DERR_KV_RANGE);
    s.len = s.len < 0 ? 0 : (int)room;
  }
  s.ql = p.q_len != nullptr ? max(0, min(p.Lq, p.q_len[b])) : p.Lq;
  const int i0 = r0 / p.G, i1 = min((r0 + n - 1) / p.G, s.ql - 1);
  s.lo = s.pos(i0, p.causal);
  s.hi = s.pos(i1, p.causal);
  s.sink = s.first = s.count = 0;
  s.per = p.per;
  if (i0 > i1 || s.hi < 0) return s;
  if (p.window > 0) {
    s.first = max(0, s.lo - p.window + 1) / kUnit;
    s.sink = min((p.sinks + kUnit - 1) / kUnit, s.first);
  }
  s.count = s.sink + s.hi / kUnit - s.first + 1;
  s.per = max(p.per, (s.count + p.parts - 1) / p.parts);
  return s;
}

__device__ __forceinline__ void mma16n8(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One unit's codes and scales in a lane's registers: two tiles of 16 keys.
template <int BITS>
struct UnitRegs {
  uint4 k[2][BITS / 4], v[2][BITS / 4], s[2];
};

template <int BITS>
__device__ __forceinline__ void load_unit(const uint8_t* blk, int half, int lane, UnitRegs<BITS>& u) {
  using B = Block<BITS>;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tile = 2 * half + i;
    const uint8_t* kb = blk + tile * B::kTileCodes + lane * 16;
    const uint8_t* vb = blk + B::kValues + tile * B::kTileCodes + (lane & 3) * 128 + (lane >> 2) * 16;
#pragma unroll
    for (int x = 0; x < BITS / 4; ++x) {
      u.k[i][x] = ld_stream(kb + x * 512);
      u.v[i][x] = ld_stream(vb + x * 512);
    }
    u.s[i] = ld_stream(blk + B::kScales + tile * 128 + (lane >> 2) * 16);
  }
}

// The lane's operand registers of one tile's keys for the two groups of dims:
// a[group][k-step][4] (rows g, g + 8; dims pairs).
template <int BITS>
__device__ __forceinline__ void key_operand(const uint4* c, int grp, uint32_t (*a)[4]) {
  uint32_t lo[4], hi[4];  // token 4q+b (row g), token 4q+b+2 (row g + 8)
  if (BITS == 4) {
    codes4(grp == 0 ? c[0].x : c[0].y, lo);
    codes4(grp == 0 ? c[0].z : c[0].w, hi);
  } else {
    const uint4 w = c[grp];
    codes8(w.x, lo);
    codes8(w.y, lo + 2);
    codes8(w.z, hi);
    codes8(w.w, hi + 2);
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
__device__ __forceinline__ void value_operand(const uint4* c, int grp, uint32_t (*a)[4]) {
  const uint4 w = c[BITS == 4 ? 0 : grp];
  const uint32_t e01 = __byte_perm(w.x, w.y, 0x5410), o01 = __byte_perm(w.x, w.y, 0x7632);
  const uint32_t e23 = __byte_perm(w.z, w.w, 0x5410), o23 = __byte_perm(w.z, w.w, 0x7632);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (BITS == 4) {
      const int sh = 8 * grp + 4 * m;
      a[m][0] = as_u32(__hsub2(as_bf2(lop_and_or(e01 >> sh, 0x000F000Fu, 0x43004300u)), as_bf2(0x43084308u)));
      a[m][1] = as_u32(__hsub2(as_bf2(lop_and_or(o01 >> sh, 0x000F000Fu, 0x43004300u)), as_bf2(0x43084308u)));
      a[m][2] = as_u32(__hsub2(as_bf2(lop_and_or(e23 >> sh, 0x000F000Fu, 0x43004300u)), as_bf2(0x43084308u)));
      a[m][3] = as_u32(__hsub2(as_bf2(lop_and_or(o23 >> sh, 0x000F000Fu, 0x43004300u)), as_bf2(0x43084308u)));
    }
  }
  if (BITS == 8) {
    uint32_t x[4][2];
    codes8(e01, x[0]);
    codes8(o01, x[1]);
    codes8(e23, x[2]);
    codes8(o23, x[3]);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[m][i] = x[i][m];
    }
  }
}

constexpr int kWarps = 4;

// One CTA per (part, kv head, row block, sequence): its warps take the part's
// units in turn, each with its own running maximum, sum and output, which are
// joined in shared memory at the end.
template <int BITS, int NT>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(AttnParams p) {
  pdl_prologue();
  constexpr int R = 8 * NT;
  __shared__ float sO[kWarps][R][HD + 4];
  __shared__ float sM[kWarps][R], sL[kWarps][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int x = blockIdx.x;  // kv head, part, row block, sequence
  const int h = x % p.c.kv_heads;
  x /= p.c.kv_heads;
  const int part = x % p.parts;
  x /= p.parts;
  const int rb = x % p.row_blocks, b = x / p.row_blocks;
  const int rows = p.Lq * p.G, r0 = rb * R;
  const Span sp = span_of(p, b, r0, R);
  const int u0 = part * sp.per, u1 = min(sp.count, u0 + sp.per);
  if (part > 0 && u0 >= sp.count) return;  // part 0 writes the rows that see nothing

  // query operand: column g of n-tile j is row r0 + 8j + g, dims 32 grp + 8t .. + 7
  uint32_t qf[NT][2][4];
  int pos[NT][2];  // positions of the accumulator's columns 2t, 2t + 1
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
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int rc = r0 + 8 * j + 2 * t + c, ic = rc / p.G;
      pos[j][c] = rc < rows && ic < sp.ql ? sp.pos(ic, p.causal) : -1;
    }
  }

  float o[NT][4][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    m[j][0] = m[j][1] = -INFINITY;
    l[j][0] = l[j][1] = 0.f;
  }
  const float grow = 8.f / p.scale_log2;  // the maximum moves in steps above 2^8 only

  auto block = [&](int u) -> const uint8_t* {
    return u < u1 ? block_of<BITS>(p.c, b, sp.unit(u) >> 1, h) : nullptr;
  };
  UnitRegs<BITS> cur;
  const uint8_t* blk = block(u0 + warp);
  if (blk) load_unit<BITS>(blk, sp.unit(u0 + warp) & 1, lane, cur);
#pragma unroll 1
  for (int u = u0 + warp; u < u1; u += kWarps) {
    const uint8_t* nblk = block(u + kWarps);
    UnitRegs<BITS> nxt;
    if (nblk) load_unit<BITS>(nblk, sp.unit(u + kWarps) & 1, lane, nxt);
    if (blk) {
      const int key0 = sp.unit(u) * kUnit;
      float s[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float s1[NT][4];
        uint32_t a[2][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][j][e] = s1[j][e] = 0.f;
        }
        key_operand<BITS>(cur.k[i], 0, a);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma16n8(s[i][j], a[0], qf[j][0][0], qf[j][0][1]);
          mma16n8(s[i][j], a[1], qf[j][0][2], qf[j][0][3]);
        }
        key_operand<BITS>(cur.k[i], 1, a);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma16n8(s1[j], a[0], qf[j][1][0], qf[j][1][1]);
          mma16n8(s1[j], a[1], qf[j][1][2], qf[j][1][3]);
        }
        const float da0 = __uint_as_float(cur.s[i].x << 16), da1 = __uint_as_float(cur.s[i].x & 0xFFFF0000u);
        const float db0 = __uint_as_float(cur.s[i].z << 16), db1 = __uint_as_float(cur.s[i].z & 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          s[i][j][0] = fmaf(s[i][j][0], da0, s1[j][0] * da1);
          s[i][j][1] = fmaf(s[i][j][1], da0, s1[j][1] * da1);
          s[i][j][2] = fmaf(s[i][j][2], db0, s1[j][2] * db1);
          s[i][j][3] = fmaf(s[i][j][3], db0, s1[j][3] * db1);
        }
      }
      // keys that a row does not see; `seen` bit (i, j, e)
      const bool inside = key0 + kUnit - 1 <= sp.lo &&
                          (p.window <= 0 || key0 > sp.hi - p.window || key0 + kUnit <= p.sinks);
      uint32_t hidden[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) hidden[j] = 0u;
      if (!inside) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int ka = key0 + i * 16 + 4 * (g >> 1) + (g & 1);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = ka + (e & 2), at = pos[j][e & 1];
              const bool sees = key <= at && (p.window <= 0 || key > at - p.window || key < p.sinks);
              if (!sees) {
                hidden[j] |= 1u << (4 * i + e);
                s[i][j][e] = -INFINITY;
              }
            }
          }
        }
      }
      bool moves = false;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float top = fmaxf(fmaxf(s[0][j][c], s[0][j][c + 2]), fmaxf(s[1][j][c], s[1][j][c + 2]));
          moves |= top > m[j][c] + grow || (m[j][c] == -INFINITY && top > -INFINITY);
        }
      }
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(fmaxf(s[0][j][c], s[0][j][c + 2]), fmaxf(s[1][j][c], s[1][j][c + 2]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float to = fmaxf(m[j][c], top);
            const float f = to == m[j][c] ? 1.f : ex2((m[j][c] - to) * p.scale_log2);
            m[j][c] = to;
            l[j][c] *= f;
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
        uint32_t b0[NT][2], b1[NT][2];
        const float va0 = __uint_as_float(cur.s[i].y << 16), va1 = __uint_as_float(cur.s[i].y & 0xFFFF0000u);
        const float vb0 = __uint_as_float(cur.s[i].w << 16), vb1 = __uint_as_float(cur.s[i].w & 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float e[4], x0[4], x1[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float mc = m[j][c & 1];
            e[c] = ex2(fmaf(s[i][j][c], p.scale_log2, mc == -INFINITY ? 0.f : -mc * p.scale_log2));
            const bool off = (hidden[j] >> (4 * i + c)) & 1u;
            l[j][c & 1] += e[c];
            x0[c] = off ? 0.f : e[c] * (c < 2 ? va0 : vb0);
            x1[c] = off ? 0.f : e[c] * (c < 2 ? va1 : vb1);
          }
          // P^T rounded to bf16 with its value scales (2^-9 of each term, as bf16 values have)
          b0[j][0] = transpose8(pack_bf16x2(x0[0], x0[1]));
          b1[j][0] = transpose8(pack_bf16x2(x0[2], x0[3]));
          b0[j][1] = transpose8(pack_bf16x2(x1[0], x1[1]));
          b1[j][1] = transpose8(pack_bf16x2(x1[2], x1[3]));
        }
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          uint32_t a[2][4];
          value_operand<BITS>(cur.v[i], grp, a);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma16n8(o[j][2 * grp], a[0], b0[j][grp], b1[j][grp]);
            mma16n8(o[j][2 * grp + 1], a[1], b0[j][grp], b1[j][grp]);
          }
        }
      }
    }
    cur = nxt;
    blk = nblk;
  }

  // join the warps: columns 2t, 2t+1 of n-tile j are rows 8j + 2t (+ 1); piece
  // 2 grp + n holds dims 32 grp + 4g + 2n and that + 1
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = l[j][c];
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
  const bool whole = sp.count <= sp.per;  // the only part of these rows
  const long long slot = (((long long)b * p.row_blocks + rb) * p.c.kv_heads + h) * p.parts + part;
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
}

// Joins the parts of a block of rows in their order: one warp per row, two dims
// per lane.
template <int NT>
__global__ void __launch_bounds__(256) join_kernel(AttnParams p) {
  pdl_prologue();
  constexpr int R = 8 * NT;
  int x = blockIdx.x;
  const int h = x % p.c.kv_heads;
  x /= p.c.kv_heads;
  const int rb = x % p.row_blocks, b = x / p.row_blocks;
  const int rows = p.Lq * p.G, r0 = rb * R;
  const Span sp = span_of(p, b, r0, R);
  if (sp.count <= sp.per) return;  // written whole
  const int n = (sp.count + sp.per - 1) / sp.per;
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < R && r0 + r < rows; r += 8) {
    const int row = r0 + r, i = row / p.G, head = h * p.G + row - i * p.G;
    const long long slot = (((long long)b * p.row_blocks + rb) * p.c.kv_heads + h) * p.parts;
    float top = -INFINITY;
    for (int y = 0; y < n; ++y) top = fmaxf(top, p.part_ml[((slot + y) * R + r) * 2]);
    float sum = 0.f, a0 = 0.f, a1 = 0.f;
    for (int y = 0; y < n; ++y) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + ((slot + y) * R + r) * 2);
      const float f = ml.x == -INFINITY ? 0.f : ex2((ml.x - top) * p.scale_log2);
      const float2 v = *reinterpret_cast<const float2*>(p.part_o + ((slot + y) * R + r) * HD + 2 * lane);
      sum += ml.x == -INFINITY ? ml.y : f * ml.y;
      a0 += f * v.x;
      a1 += f * v.y;
    }
    const bool empty = i >= sp.ql || sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    const uint32_t out = empty ? 0u : pack_bf16x2(a0 * inv, a1 * inv);
    *reinterpret_cast<uint32_t*>(p.o + (long long)b * p.o_batch + (long long)i * p.o_row + (long long)head * HD +
                                 2 * lane) = out;
  }
}

}  // namespace kv
}  // namespace vla
