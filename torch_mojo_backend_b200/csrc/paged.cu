// The paged key/value cache: appending new tokens, attention of the newest tokens over the pages, reading sequences back.
//
// A cache is a pool of pages, each `page_size` tokens of every KV head, (pages, Hkv, page_size, D); a row of the block table
// names the pages of a sequence in order.  Pages hold the 16-bit type itself, or 4 bits an element: codes 0..15, and for every
// 32 elements a scale and a minimum of the 16-bit type; an element is code * scale + minimum.  The codes of a row lie in the
// order the attention kernel's fragments want them in:
//   * keys:   the 32-bit word of (t, G), t = 0..3, is word t * (D / 32) + G of the row and holds elements 32 G + 8 t + 0..7, the
//             first in the lowest bits: thread t of a quad reads D / 8 contiguous bytes, one word of every group G;
//   * values: the 16 bits of (g, G), g = 0..7, are halfword g * (D / 32) + G and hold elements 32 G + 4 g + 0..3: lane group g
//             reads D / 16 contiguous bytes, and the elements of a tensor-core tile share a group, that is a scale.
//
// Every index that comes from device memory (pages, lengths, positions) is checked before it is used.  What depends on a bad one
// is not written (append) or is NaN (attention, reading back), and the status word says so.
#include <algorithm>
#include <cmath>
#include <mutex>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/b200fa.h"
#include "common.cuh"
#include "ptx.cuh"

namespace b200fa {
namespace {

constexpr int kGroup = 32;   // elements that share a scale and a minimum

__device__ __forceinline__ void report_bad_index(uint32_t* status, uint32_t site) {
  if (status) atomicCAS(status, kStatusOk, kStatusBadIndex | site);
}

// Tokens of a sequence: `len` in the cache, the last `n` of them new; false if the numbers cannot be.
struct Sequence {
  int len, n;
};
__device__ __forceinline__ bool sequence_of(const PagedCache& c, int b, int S, Sequence* s) {
  s->len = __ldg(c.lengths + b);
  s->n = c.new_lengths ? __ldg(c.new_lengths + b) : S;
  return s->len >= 0 && s->len <= c.capacity && s->n >= 0 && s->n <= S;
}

__device__ __forceinline__ float lo_f32(uint32_t w, __nv_bfloat16) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(uint32_t w, __nv_bfloat16) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float lo_f32(uint32_t w, __half) { return __half2float(__ushort_as_half(static_cast<unsigned short>(w))); }
__device__ __forceinline__ float hi_f32(uint32_t w, __half) { return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16))); }
template <typename T>
__device__ __forceinline__ uint32_t pack_t(float lo, float hi) {
  return pack2<sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value>(lo, hi);
}
template <typename T>
__device__ __forceinline__ float round_t(float x) { return lo_f32(pack_t<T>(x, 0.f), T()); }

template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const T2 r = __hmin2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const T2 r = __hmax2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// ------------------------------------------------------------------------------------------
// Append.  D / 8 lanes take a row (16 bytes each), one head's query, key or value of one token, and a warp kChunk heads of the
// queries, keys or values of one token, kRows of them in each thread: the token's place and angles are looked up once, and the loads of all its rows are in
// flight together.  With (a, b) a pair of elements that turn together (i and i + R / 2, or 2 i and 2 i + 1, of the first R) and
// (c, s) its position's cos and sin, a' = a c - b s, b' = b c + a s: every product and sum rounded to fp32 on its own (no FMA),
// then to the type, so that the results are those of the formula in fp32 whatever computes it.  Copy-bound: each element is
// read and written once.  A row of 4 bits: scale = (max - min) / 15 rounded to the type, code = round((x - min) / scale), of the
// elements as rounded to the type.  Where an element of a group is not finite the scale is NaN, and so is the group.
// B200, one row a thread / this: 6 prompts of up to 1500 tokens, 16 + 4 heads, D = 64, 4 bits: 21 / 12-13 us, most of it by the
// reciprocal; 64 single tokens, 32 + 8 heads, D = 128, 16 bits: 2.4 us.
// ------------------------------------------------------------------------------------------
template <typename T, int kD>
struct AppendCfg {
  static constexpr int kLanes = kD / 8, kSide = 32 / kLanes;   // rows side by side
  static constexpr int kRows = 4, kChunk = kRows * kSide;
};

// kClear: rows of q_out that no new token has are written too.  (Asked at run time it takes 8 registers, an eighth of the blocks of an SM and
// 4 % of the time of the prompts above from all other calls.)
template <typename T, int kD, int kBits, bool kInterleaved, bool kClear>
__global__ void __launch_bounds__(128) paged_append_kernel(const AppendParams p) {
  using Cfg = AppendCfg<T, kD>;
  constexpr int kLanes = Cfg::kLanes;
  constexpr unsigned kFull = 0xffffffffu;
  const int lane = threadIdx.x & 31, li = lane % kLanes;
  // the warp's token, and its kChunk heads of q, k or v
  const int of_q = (p.Hq + Cfg::kChunk - 1) / Cfg::kChunk, of_k = (p.c.Hkv + Cfg::kChunk - 1) / Cfg::kChunk;
  const unsigned item = blockIdx.x * 4 + static_cast<unsigned>(warp_index());
  const unsigned token = item / (of_q + 2 * of_k);
  int chunk = static_cast<int>(item - token * (of_q + 2 * of_k));
  const int what = chunk < of_q ? 0 : chunk < of_q + of_k ? 1 : 2;
  chunk -= what == 0 ? 0 : what == 1 ? of_q : of_q + of_k;
  const int b = static_cast<int>(token / p.S), s = static_cast<int>(token - static_cast<unsigned>(b) * p.S);
  if (b >= p.c.B) return;
  const int heads = what == 0 ? p.Hq : p.c.Hkv, h0 = chunk * Cfg::kChunk + lane / kLanes;
  const View4& from = what == 0 ? p.q : what == 1 ? p.k : p.v;
  const T* src = reinterpret_cast<const T*>(from.ptr) + static_cast<int64_t>(b) * from.sb + static_cast<int64_t>(h0) * from.sh +
                 static_cast<int64_t>(s) * from.ss + li * 8;
  uint4 x[Cfg::kRows];
#pragma unroll
  for (int u = 0; u < Cfg::kRows; ++u)
    x[u] = h0 + u * Cfg::kSide < heads ? __ldg(reinterpret_cast<const uint4*>(src + u * Cfg::kSide * from.sh)) : make_uint4(0, 0, 0, 0);
  Sequence seq;
  const bool good = sequence_of(p.c, b, p.S, &seq);
  const int pos = seq.len - seq.n + s;
  auto q_row = [&](int u) {   // (if what == 0)
    return reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out.ptr) + static_cast<int64_t>(b) * p.q_out.sb +
                                    static_cast<int64_t>(h0 + u * Cfg::kSide) * p.q_out.sh + static_cast<int64_t>(s) * p.q_out.ss + li * 8);
  };
  auto clear = [&](uint32_t word) {   // the rows of queries that are not turned
    if (!kClear || what != 0) return;
#pragma unroll 1
    for (int u = 0; u < Cfg::kRows; ++u)
      if (h0 + u * Cfg::kSide < heads) *q_row(u) = make_uint4(word, word, word, word);
  };
  constexpr uint32_t kNaN2 = 0x7fff7fffu;   // in either type
  if (!good) {
    if (lane == 0) report_bad_index(p.c.status, 1);
    return clear(kNaN2);
  }
  if (s >= seq.n || pos < 0) return clear(0);
  if (p.rotary != 0 && pos >= p.positions) {
    if (lane == 0) report_bad_index(p.c.status, 2);
    return clear(kNaN2);
  }
  uint32_t row0 = 0;   // of head h0 in the pages
  if (what != 0) {
    const int page = __ldg(p.c.table + static_cast<int64_t>(b) * p.c.table_stride + (pos >> p.c.shift));
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.pages)) {
      if (lane == 0) report_bad_index(p.c.status, 3);
      return;
    }
    row0 = (static_cast<uint32_t>(page * p.c.Hkv + h0) << p.c.shift) + (pos & ((1 << p.c.shift) - 1));
  }
  const int e0 = li * 8, half = p.rotary / 2;
  const bool first = e0 < half;
  constexpr int kAngles = kInterleaved ? 4 : 8;
  float cs[kAngles], sn[kAngles];
  if (what != 2 && e0 < p.rotary) {
    const int64_t angle = static_cast<int64_t>(pos) * half + (kInterleaved ? e0 / 2 : first ? e0 : e0 - half);
#pragma unroll
    for (int i = 0; i < kAngles / 4; ++i) {
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos + angle) + i), s4 = __ldg(reinterpret_cast<const float4*>(p.sin + angle) + i);
      cs[4 * i] = c4.x; cs[4 * i + 1] = c4.y; cs[4 * i + 2] = c4.z; cs[4 * i + 3] = c4.w;
      sn[4 * i] = s4.x; sn[4 * i + 1] = s4.y; sn[4 * i + 2] = s4.z; sn[4 * i + 3] = s4.w;
    }
  }
#pragma unroll
  for (int u = 0; u < Cfg::kRows; ++u) {
    if (chunk * Cfg::kChunk + u * Cfg::kSide >= heads) break;
    const bool write = h0 + u * Cfg::kSide < heads;
    uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    if (p.rotary && what != 2) {
      const bool turn = e0 < p.rotary;
      if constexpr (kInterleaved) {
        if (turn) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = lo_f32(w[i], T()), d = hi_f32(w[i], T());
            w[i] = pack_t<T>(__fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(d, sn[i])), __fadd_rn(__fmul_rn(d, cs[i]), __fmul_rn(a, sn[i])));
          }
        }
      } else {
        // the other elements of the pairs are half / 8 lanes away
        const int from = e0 < p.rotary ? (first ? lane + half / 8 : lane - half / 8) : lane;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(kFull, w[i], from);
        if (turn) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float a = j ? hi_f32(w[i], T()) : lo_f32(w[i], T()), d = j ? hi_f32(o[i], T()) : lo_f32(o[i], T());
              const float ac = __fmul_rn(a, cs[2 * i + j]), ds = __fmul_rn(d, sn[2 * i + j]);
              y[j] = first ? __fsub_rn(ac, ds) : __fadd_rn(ac, ds);
            }
            w[i] = pack_t<T>(y[0], y[1]);
          }
        }
      }
    }
    if (what == 0) {
      if (write) *q_row(u) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
    }
    const uint64_t at = row0 + (static_cast<uint32_t>(u * Cfg::kSide) << p.c.shift);   // the row in the pages
    if constexpr (kBits == 16) {
      if (write) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(what == 1 ? p.c.k : p.c.v) + at * kD + li * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      // the four lanes of a group find its minimum and maximum, two elements at a time
      uint32_t lo2 = min2<T>(min2<T>(w[0], w[1]), min2<T>(w[2], w[3])), hi2 = max2<T>(max2<T>(w[0], w[1]), max2<T>(w[2], w[3]));
#pragma unroll
      for (int off = 1; off <= 2; off <<= 1) {
        lo2 = min2<T>(lo2, __shfl_xor_sync(kFull, lo2, off));
        hi2 = max2<T>(hi2, __shfl_xor_sync(kFull, hi2, off));
      }
      float v[8], odd = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = i & 1 ? hi_f32(w[i >> 1], T()) : lo_f32(w[i >> 1], T());
        odd = fmaf(v[i], 0.f, odd);   // NaN if an element is not finite
      }
      const unsigned odd_lanes = __ballot_sync(kFull, odd != 0.f);
      if (!write) continue;   // (nothing below needs the other lanes; the next row's shuffles wait for all)
      const float low = fminf(lo_f32(lo2, T()), hi_f32(lo2, T())), high = fmaxf(lo_f32(hi2, T()), hi_f32(hi2, T()));
      float scale = round_t<T>(__fdiv_rn(__fsub_rn(high, low), 15.f));
      if ((odd_lanes >> (lane & ~3)) & 15u) scale = __uint_as_float(0x7fffffffu);
      // round((x - low) / scale), the division rounded to nearest, at most 15.  The product with the reciprocal is within 3e-6 of
      // that quotient and rounds as it does unless it is that near to a half; then the division decides.  (A division for each
      // element was most of the kernel's instructions.)
      const float inverse = __fdiv_rn(1.f, scale);
      const bool tiny = !(scale >= 1e-37f);   // (its reciprocal may be infinite)
      uint32_t codes = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        constexpr float kInts = 12582912.f;   // 1.5 * 2^23: the sum's last bits are the rounded number
        const float d = __fsub_rn(v[i], low);
        float q = fminf(__fmul_rn(d, inverse), 15.f), r = __fadd_rn(q, kInts);
        if (tiny || !(fabsf(q - __fsub_rn(r, kInts)) < 0.4999f)) r = __fadd_rn(fminf(__fdiv_rn(d, scale), 15.f), kInts);
        codes |= (__float_as_uint(r) & 15u) << (4 * i);
      }
      if (!(scale > 0.f)) codes = 0;
      const int G = li >> 2, t = li & 3;
      constexpr int kGroups = kD / kGroup;
      uint32_t* row_words = reinterpret_cast<uint32_t*>(what == 1 ? p.c.k : p.c.v) + at * (kD / 8);
      if (what == 1) {
        row_words[t * kGroups + G] = codes;
      } else {
        uint16_t* halves = reinterpret_cast<uint16_t*>(row_words);
        halves[2 * t * kGroups + G] = static_cast<uint16_t>(codes);
        halves[(2 * t + 1) * kGroups + G] = static_cast<uint16_t>(codes >> 16);
      }
      if (t == 0) {
        uint32_t* scales = reinterpret_cast<uint32_t*>(what == 1 ? p.c.k_scales : p.c.v_scales) + at * kGroups;
        scales[G] = pack_t<T>(scale, low);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// Reading back.  D / 8 lanes take a row of k and the same row of v; rows behind a sequence's last are zero.  Copy-bound:
// four sequences of up to 16896 tokens, 8 KV heads, D = 128, 16 bits: 84 us, 6.3 TB/s of what is read and written.
// ------------------------------------------------------------------------------------------
template <typename T, int kD, int kBits>
__global__ void __launch_bounds__(256) paged_gather_kernel(const GatherParams p) {
  constexpr int kLanes = kD / 8, kGroups = kD / kGroup;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int li = static_cast<int>(threadIdx.x) % kLanes;
  const int64_t row = idx / kLanes;   // (batch, head, token)
  const int64_t bh = row / p.S;
  const int b = static_cast<int>(bh / p.c.Hkv), h = static_cast<int>(bh - static_cast<int64_t>(b) * p.c.Hkv);
  const int s = static_cast<int>(row - bh * p.S);
  if (b >= p.c.B) return;
  const int len = __ldg(p.c.lengths + b);
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  const bool bad_len = len < 0 || len > p.c.capacity;
  int page = -1;
  if (!bad_len && s < len) page = __ldg(p.c.table + static_cast<int64_t>(b) * p.c.table_stride + (s >> p.c.shift));
  if (bad_len || (s < len && static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.pages))) {
    if (li == 0) report_bad_index(p.c.status, bad_len ? 4 : 5);
    k.x = k.y = k.z = k.w = 0x7fff7fffu;   // NaN in either type
    v = k;
  } else if (s < len) {
    const int64_t at = ((static_cast<int64_t>(page) * p.c.Hkv + h) << p.c.shift) + (s & ((1 << p.c.shift) - 1));
    if constexpr (kBits == 16) {
      k = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.c.k) + at * kD) + li);
      v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.c.v) + at * kD) + li);
    } else {
      const int G = li >> 2, t = li & 3;
      const uint32_t ck = __ldg(reinterpret_cast<const uint32_t*>(p.c.k) + at * (kD / 8) + t * kGroups + G);
      const uint16_t* halves = reinterpret_cast<const uint16_t*>(p.c.v) + at * (kD / 4);
      const uint32_t cv = __ldg(halves + 2 * t * kGroups + G) | static_cast<uint32_t>(__ldg(halves + (2 * t + 1) * kGroups + G)) << 16;
      const uint32_t sk = __ldg(reinterpret_cast<const uint32_t*>(p.c.k_scales) + at * kGroups + G);
      const uint32_t sv = __ldg(reinterpret_cast<const uint32_t*>(p.c.v_scales) + at * kGroups + G);
      auto value = [](uint32_t codes, int i, uint32_t sc) {
        return __fadd_rn(__fmul_rn(static_cast<float>((codes >> (4 * i)) & 15u), lo_f32(sc, T())), hi_f32(sc, T()));
      };
      uint32_t wk[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        wk[i] = pack_t<T>(value(ck, 2 * i, sk), value(ck, 2 * i + 1, sk));
        wv[i] = pack_t<T>(value(cv, 2 * i, sv), value(cv, 2 * i + 1, sv));
      }
      k = make_uint4(wk[0], wk[1], wk[2], wk[3]);
      v = make_uint4(wv[0], wv[1], wv[2], wv[3]);
    }
  }
  auto store = [&](const View4& t, const uint4& x) {
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(t.ptr) + static_cast<int64_t>(b) * t.sb + static_cast<int64_t>(h) * t.sh +
                              static_cast<int64_t>(s) * t.ss + li * 8) = x;
  };
  store(p.k, k);
  store(p.v, v);
}

// ------------------------------------------------------------------------------------------
// Attention.  A unit is one KV head of one sequence and up to 8 kNT query rows (new tokens x query heads of the group, token by
// token); a cluster of blocks shares its keys and merges (max, sum, O) through distributed shared memory.  A warp takes 16 keys at a
// time (4 bits: two such halves a step), all in one page: S^T = K Q^T and O^T += V^T P^T by mma.sync m16n8k16, keys and then head-dim elements the M dimension,
// rows the N dimension, operands from global memory to fragment registers directly.  HBM-bound by design: K and V are read
// once per unit.  Thread (g, t) = (lane / 4, lane % 4) owns keys g and g + 8 and rows 2t and 2t + 1 of each tile in the softmax.
//   * 16 bits: K as thread (g, t) reads 16 bytes at (4i + t) 16 of key rows g and g + 8 (any permutation of the contraction
//     index will do if Q has the same); V as it reads 16 bytes at 128 h + 16 g of rows 2t, 2t+1, 2t+8, 2t+9, whose registers a
//     byte permute turns into (key, key + 1) pairs.
//   * 4 bits: the codes are operands, the scales stay out of the products.  S = sum over groups G of ks_G (q_G . c_G) +
//     km_G sum(q_G), with the codes as fp16 and q as fp16, a row of it multiplied by the power of two that brings its largest
//     element to 1..2 (exact but for elements below 2^-14 of that one, which are off by 2^-25 of it); sum over G of km_G sum(q_G) is
//     one more product, keys by groups, of sum(q_G) in three parts of the type.  O_G = sum over keys of (P vs_G) (c - 8) +
//     P (vm_G + 8 vs_G): P vs_G is the B operand, rounded to the cache's type, c - 8 is exact, and the second sum, the same for
//     the 32 elements of a group, is one product as well, (vs, vm) of the groups by keys times P as rounded to the type.  (Codes of
//     0..15 instead would make both sums several times their difference, and the rounding of P vs_G with them.)
// The row maximum moves only when a score exceeds it by 2^8 (a vote per step instead of six shuffles), so P is at most 256; at
// most 4 where P vs_G is an fp16, whose largest scale is 8734.
// B200, decode of one token, 8 KV heads, groups of 4, D = 128, bf16: 8 sequences of up to 32768 keys (spread 60 %), 16 bits: 136 us,
// 0.89 of the copy rate; 16 of up to 32768 (spread 30 %), 4 bits: 170-174 us, 0.51-0.52 of it.  The 4-bit kernel is bound by issue:
// about 420 instructions for 16 keys of a head, 61 % of the issue slots and the logic unit at 59 % of its peak while an SM is busy, which is
// 80 % of the time.  (16 bits by bulk copies into rings: no better.)
// Keys that no row of the unit sees are never read, not even into a product with zero: their places in a step re-read a key that is
// seen (pages behind a window may have been given to another sequence).
// ------------------------------------------------------------------------------------------
constexpr int kStepKeys = 16;
constexpr int kMaxPeers = 16;

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// The codes of a word (four in each half) as four pairs, one from each half, of the same place, less `minus` (0 or 8).  The logic
// unit, at half the rate of the others, binds the unpacking.  An fp16 1024 has ten mantissa bits below it: codes at bits 0..3 or
// 4..7 make 1024 + c and 1024 + 16 c, and a half-precision FMA takes the rest off, exactly: five logic instructions a word.  A
// bf16 128 has seven, which take one code: seven instructions a word.
// `one`: the 1024 or 128 in both halves, kOneF16 or kOneBf16, from the launch: the compiler makes two instructions of a mask and a
// bit pattern that it knows, since one takes one immediate.
constexpr uint32_t kOneF16 = 0x64006400u, kOneBf16 = 0x43004300u;
__device__ __forceinline__ uint32_t masked_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));   // (w & mask) | bits
  return r;
}
template <typename T>
__device__ __forceinline__ void codes_of(uint32_t w, float minus, uint32_t one, uint32_t (&c)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t w8 = w >> 8;
    c[0] = masked_or(w, 0x000f000fu, one);
    c[1] = masked_or(w, 0x00f000f0u, one);
    c[2] = masked_or(w8, 0x000f000fu, one);
    c[3] = masked_or(w8, 0x00f000f0u, one);
    const __half2 lo = __float2half2_rn(-1024.f - minus), hi = __float2half2_rn(-64.f - minus), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 x = *reinterpret_cast<const __half2*>(&c[j]);
      const __half2 y = j & 1 ? __hfma2(x, sixteenth, hi) : __hadd2(x, lo);
      c[j] = *reinterpret_cast<const uint32_t*>(&y);
    }
  } else {
    const __nv_bfloat162 off = __float2bfloat162_rn(-128.f - minus);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = masked_or(w >> (4 * j), 0x000f000fu, one);
      const __nv_bfloat162 y = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&c[j]), off);
      c[j] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
}

// The rows and keys of one unit, as a block sees them.
struct Unit {
  int b, hk, rank;                   // sequence, KV head, place in the cluster
  unsigned part;                     // the cluster's number among those of all units, team by team
  int row0, rows, group;             // rows row0 .. row0 + rows - 1 of the group's (new tokens x query heads)
  int first_pos, p_first, p_last;    // positions of the first new token, of the unit's first row and of its last
  KeyBlocks list;                    // steps of keys
  int hidden_from, hidden_to;        // keys between the sinks and the first row's window
  int low;                           // a step that begins at or below it holds keys ahead of some row's window; -1 without one
  int begin, end;                    // the block's share of the steps
  bool good;                         // the sequence's numbers can be
};
template <int kKeys>
__device__ __forceinline__ Unit unit_of(const AttendParams& p, int max_rows) {
  Unit u;
  u.b = blockIdx.z;
  u.hk = blockIdx.y;
  const unsigned shares = p.peers * p.teams, tile = blockIdx.x / shares, share = blockIdx.x - tile * shares;
  const unsigned team = share / static_cast<unsigned>(p.peers), tiles = gridDim.x / shares;
  u.rank = share - team * p.peers;
  u.part = ((blockIdx.z * gridDim.y + blockIdx.y) * tiles + tile) * p.teams + team;
  u.row0 = tile * max_rows;
  u.group = p.group;
  Sequence seq;
  u.good = sequence_of(p.c, u.b, p.S, &seq);
  if (!u.good) {   // every row of the sequence is NaN
    if (threadIdx.x == 0) report_bad_index(p.c.status, 6);
    seq.len = 0;
    seq.n = p.S;
  }
  u.rows = min(max_rows, seq.n * u.group - u.row0);
  u.first_pos = seq.len - seq.n;   // negative: the token sees nothing
  u.p_first = u.first_pos + u.row0 / u.group;
  u.p_last = u.first_pos + (u.row0 + max(u.rows, 1) - 1) / u.group;
  u.list = KeyBlocks{0, 0, max(0, u.p_last + kKeys) / kKeys};
  u.hidden_from = u.hidden_to = 0;
  u.low = -1;
  if (p.window) {
    u.list = window_blocks<kKeys>(u.p_first, u.p_last, seq.len, p.window, p.sinks);
    u.hidden_from = p.sinks;
    u.hidden_to = u.p_first - p.window + 1;
    u.low = u.p_last - p.window;
  }
  // (at most 2^20 steps and 256 shares)
  u.begin = static_cast<int>(static_cast<unsigned>(u.list.n * share) / shares);
  u.end = static_cast<int>(static_cast<unsigned>(u.list.n * (share + 1)) / shares);
  return u;
}
// place in a step of the key that is read for key `k` of it
template <int kKeys>
__device__ __forceinline__ int place(const Unit& u, int base, int k) {
  int key = min(base + k, u.p_last);
  if (key >= u.hidden_from && key < u.hidden_to) key = u.hidden_to < base + kKeys ? u.hidden_to : u.hidden_from - 1;
  return key - base;
}
// every key of the step is one that some row sees
template <int kKeys>
__device__ __forceinline__ bool whole_step(const Unit& u, int base) {
  return base + kKeys - 1 <= u.p_last && (base >= u.hidden_to || base + kKeys - 1 < u.hidden_from);
}
// some key of the step is one that some row does not see
template <int kKeys>
__device__ __forceinline__ bool edge_step(const Unit& u, const AttendParams& p, int base) {
  return base + kKeys - 1 > u.p_first || (base <= u.low && base + kKeys - 1 >= p.sinks);
}
template <typename T>
__device__ __forceinline__ const T* query_row(const AttendParams& p, const Unit& u, int r) {
  const int s = static_cast<int>(static_cast<unsigned>(u.row0 + r) / static_cast<unsigned>(u.group)), h = u.hk * u.group + u.row0 + r - s * u.group;
  return reinterpret_cast<const T*>(p.q.ptr) + static_cast<int64_t>(u.b) * p.q.sb + static_cast<int64_t>(h) * p.q.sh + static_cast<int64_t>(s) * p.q.ss;
}
// row of the pages that holds the first key of a step, which lies in page `page`; page 0 and `bad` for one that is none
__device__ __forceinline__ uint32_t page_row(const PagedCache& c, int hk, int page, int base, bool* bad) {
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.pages)) {
    *bad = true;
    page = 0;
  }
  return (static_cast<uint32_t>(page * c.Hkv + hk) << c.shift) + (base & ((1 << c.shift) - 1));
}

// What a warp holds of its rows: thread (g, t) has rows 2t and 2t + 1 of each tile of eight.
template <int kNT, int kTiles, bool kZ>
struct RowState {
  float m[kNT][2], shift[kNT][2], limit[kNT][2], l[kNT][2];   // shift: -m, 0 as long as there is none; limit: where it moves
  float o[kNT][kTiles][4];   // O^T: [0] (slot g, row 2t) [1] (slot g, row 2t + 1) [2], [3] slot g + 8
  float z[kZ ? kNT : 1][4];  // 4 bits: sums of P vs (slots g < D / 32) and P vm (the next D / 32)
  int pos[kNT][2];           // positions of the rows (of those behind the last, too, which are not written)

  __device__ __forceinline__ void clear(const Unit& u, int t) {
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) pos[n][e] = u.first_pos + static_cast<int>(static_cast<unsigned>(u.row0 + 8 * n + 2 * t + e) / static_cast<unsigned>(u.group));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = limit[n][e] = -INFINITY;
        shift[n][e] = l[n][e] = 0.f;
        if (kZ) z[n][e] = z[n][2 + e] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
    }
  }
  // raises the maxima of the rows that have a score above theirs, and rescales what was summed
  template <int kH>
  __device__ __forceinline__ void raise(float (&x)[kH][kNT][4], float lazy) {
    constexpr unsigned kFull = 0xffffffffu;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(x[0][n][e], x[0][n][2 + e]);
        if (kH == 2) top = fmaxf(top, fmaxf(x[kH - 1][n][e], x[kH - 1][n][2 + e]));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 4));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 8));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 16));   // relative to the standing maximum (to 0 without one)
        const bool none = m[n][e] == -INFINITY;
        if (top > (none ? -INFINITY : 0.f)) {
          const float corr = none ? 0.f : exp2f(-top);
          m[n][e] = none ? top : m[n][e] + top;
          shift[n][e] = -m[n][e];
          limit[n][e] = lazy;
#pragma unroll
          for (int h = 0; h < kH; ++h) {
            x[h][n][e] -= top;
            x[h][n][2 + e] -= top;
          }
          l[n][e] *= corr;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            o[n][j][e] *= corr;
            o[n][j][2 + e] *= corr;
          }
          if (kZ) z[n][e] *= corr;
        }
      }
  }
  // scores less the rows' maxima, of kH times 16 keys, x[h][n][0] (key g, row 2t) [1] (key g, row 2t + 1) [2], [3] key g + 8, to
  // probabilities
  template <int kH>
  __device__ __forceinline__ void probabilities(float (&x)[kH][kNT][4], float lazy) {
    bool far = false;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(x[0][n][e], x[0][n][2 + e]);
        if (kH == 2) top = fmaxf(top, fmaxf(x[kH - 1][n][e], x[kH - 1][n][2 + e]));
        far |= top > limit[n][e];
      }
    if (__any_sync(0xffffffffu, far)) raise(x, lazy);
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int h = 0; h < kH; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h][n][e] = ex2_approx(x[h][n][e]);
        l[n][0] += x[h][n][0] + x[h][n][2];   // this thread's keys; summed over g at the end
        l[n][1] += x[h][n][1] + x[h][n][3];
      }
  }
  // -inf for the scores of keys (`first` and `second` of this thread) that a row does not see
  __device__ __forceinline__ void mask(float (&x)[kNT][4], const AttendParams& p, int first, int second) const {
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = e < 2 ? first : second, at = pos[n][e & 1];
        if (key > at || (p.window && key <= at - p.window && key >= p.sinks)) x[n][e] = -INFINITY;
      }
  }
};

// The last steps of a block: every warp has left its unnormalised O of row r at o + warp * stride + r * kRow, and the row's max and sum
// behind it.  They are merged in the block, then by the blocks of the cluster, each of which takes its share of the rows'
// 16-byte pieces from its peers' shared memory.  A row's weights are made once, by one thread.  (With each thread's own weights for
// each pair of elements a call of 16 keys and 16 rows on 256 KV heads took 13.9 us instead of 5.8.)  Where several clusters, `teams`,
// share a unit, each leaves its rows like a warp does, in the workspace, for paged_join_kernel.
template <int kD>
constexpr int kRow = kD + 4;   // floats: a row, its max and sum, 16-byte aligned

template <typename T>
__device__ __forceinline__ void write_row(const AttendParams& p, const Unit& u, int r, int c, float4 x) {
  const int row = u.row0 + r, s = static_cast<int>(static_cast<unsigned>(row) / static_cast<unsigned>(u.group)), h = u.hk * u.group + row - s * u.group;
  T* dst = reinterpret_cast<T*>(p.out.ptr) + static_cast<int64_t>(u.b) * p.out.sb + static_cast<int64_t>(h) * p.out.sh + static_cast<int64_t>(s) * p.out.ss + c * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_t<T>(x.x, x.y), pack_t<T>(x.z, x.w));
}
// 1 / sum, and the row's lse; a row without a key is 0 with lse -inf; a NaN stays one
__device__ __forceinline__ float finish_row(const AttendParams& p, const Unit& u, int r, float m, float l, bool lse) {
  if (lse) {
    const int row = u.row0 + r, s = static_cast<int>(static_cast<unsigned>(row) / static_cast<unsigned>(u.group)), h = u.hk * u.group + row - s * u.group;
    p.lse[(static_cast<int64_t>(u.b) * p.Hq + h) * p.S + s] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
  }
  return l == 0.f ? 0.f : 1.f / l;
}

template <typename T, int kD, int kNT, int kWarps>
__device__ __forceinline__ void merge(const AttendParams& p, const Unit& u, float* o, int stride) {
  constexpr int kPieces = kD / 4, kRows = 8 * kNT, kThreads = kWarps * 32;
  __shared__ float sWeight[kRows][kWarps > kMaxPeers ? kWarps : kMaxPeers];
  __shared__ float2 sML[kRows];
  const int tid = threadIdx.x, peers = p.peers, rank = u.rank;
  float* const part = p.teams > 1 ? p.parts + static_cast<int64_t>(u.part) * (kRows * kRow<kD>) : nullptr;   // (never with one peer)
  __syncthreads();
  if (tid < u.rows) {
    const float* row = o + tid * kRow<kD> + kD;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, row[w * stride]);
    const float m_use = m == -INFINITY ? 0.f : m;
    float weight[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      weight[w] = ex2_approx(row[w * stride] - m_use);   // 0 for a warp that saw no key of the row
      l = fmaf(row[w * stride + 1], weight[w], l);
    }
    const float inv = peers == 1 ? finish_row(p, u, tid, m, l, true) : 1.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sWeight[tid][w] = weight[w] * inv;
    sML[tid] = make_float2(m, l);
  }
  __syncthreads();
  for (int i = tid; i < u.rows * kPieces; i += kThreads) {
    const int r = i / kPieces, c = i % kPieces;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(o + w * stride + r * kRow<kD> + c * 4);
      const float a = sWeight[r][w];
      acc.x = fmaf(x.x, a, acc.x); acc.y = fmaf(x.y, a, acc.y); acc.z = fmaf(x.z, a, acc.z); acc.w = fmaf(x.w, a, acc.w);
    }
    if (peers == 1) write_row<T>(p, u, r, c, acc);
    else *reinterpret_cast<float4*>(o + r * kRow<kD> + c * 4) = acc;   // (this thread alone reads and writes the piece)
  }
  if (peers == 1) return;
  cluster_sync();
  if (tid < u.rows) {
    const uint32_t a_ml = smem_u32(sML + tid);
    float2 v[kMaxPeers];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) v[i] = i < peers ? peer_load_f32x2(a_ml, i) : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) m = fmaxf(m, v[i].x);
    const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) {
      v[i].x = ex2_approx(v[i].x - m_use);
      l = fmaf(v[i].y, v[i].x, l);
    }
    if (part && rank == 0) *reinterpret_cast<float2*>(part + tid * kRow<kD> + kD) = make_float2(m, l);
    const float inv = part ? 1.f : finish_row(p, u, tid, m, l, rank == 0);
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) sWeight[tid][i] = v[i].x * inv;
  }
  __syncthreads();
  for (int i = rank * kThreads + tid; i < u.rows * kPieces; i += peers * kThreads) {
    const int r = i / kPieces, c = i % kPieces;
    const uint32_t at = smem_u32(o + r * kRow<kD> + c * 4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int first = 0; first < kMaxPeers; first += 8) {   // eight loads in flight
      if (first >= peers) break;
      float4 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (first + j < peers) x[j] = peer_load_f32x4(at, first + j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (first + j < peers) {
          const float a = sWeight[r][first + j];
          acc.x = fmaf(x[j].x, a, acc.x); acc.y = fmaf(x[j].y, a, acc.y); acc.z = fmaf(x[j].z, a, acc.z); acc.w = fmaf(x[j].w, a, acc.w);
        }
      }
    }
    if (part) *reinterpret_cast<float4*>(part + r * kRow<kD> + c * 4) = acc;
    else write_row<T>(p, u, r, c, acc);
  }
  cluster_sync();   // no block leaves while a peer may still read its shared memory
}

// The rows of a unit from its teams' parts, in the order of the teams.  `p` has one peer and one team: a block is a unit.
constexpr int kMaxTeams = 16, kJoinThreads = 256;
template <typename T, int kD, int kRows>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const AttendParams p, const int teams) {
  constexpr int kPieces = kD / 4;
  __shared__ float2 sML[kRows][kMaxTeams];
  __shared__ float sWeight[kRows][kMaxTeams];
  const int tid = threadIdx.x;
  const Unit u = unit_of<16>(p, kRows);
  const float* const parts = p.parts + static_cast<int64_t>(u.part) * teams * (kRows * kRow<kD>);
  for (int i = tid; i < u.rows * teams; i += kJoinThreads) {
    const int r = i / teams, k = i - r * teams;
    sML[r][k] = *reinterpret_cast<const float2*>(parts + (k * kRows + r) * kRow<kD> + kD);
  }
  __syncthreads();
  if (tid < u.rows) {
    float m = -INFINITY, l = 0.f;
    for (int k = 0; k < teams; ++k) m = fmaxf(m, sML[tid][k].x);
    const float m_use = m == -INFINITY ? 0.f : m;
    for (int k = 0; k < teams; ++k) {
      const float weight = ex2_approx(sML[tid][k].x - m_use);
      l = fmaf(sML[tid][k].y, weight, l);
      sWeight[tid][k] = weight;
    }
    const float inv = finish_row(p, u, tid, m, l, true);
    for (int k = 0; k < teams; ++k) sWeight[tid][k] *= inv;
  }
  __syncthreads();
  for (int i = tid; i < u.rows * kPieces; i += kJoinThreads) {
    const int r = i / kPieces, c = i % kPieces;
    float4 x[kMaxTeams];
#pragma unroll
    for (int k = 0; k < kMaxTeams; ++k) {
      if (k < teams) x[k] = *reinterpret_cast<const float4*>(parts + (k * kRows + r) * kRow<kD> + c * 4);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kMaxTeams; ++k) {
      if (k < teams) {
        const float a = sWeight[r][k];
        acc.x = fmaf(x[k].x, a, acc.x); acc.y = fmaf(x[k].y, a, acc.y); acc.z = fmaf(x[k].z, a, acc.z); acc.w = fmaf(x[k].w, a, acc.w);
      }
    }
    write_row<T>(p, u, r, c, acc);
  }
}

// Blocks of four warps that an SM takes, by their registers; a block of `kWide` warps has an SM to itself.
template <int kD, int kNT, int kBits>
struct AttendCfg {
  static constexpr int kPerSm = kNT == 2 ? 2 : kD == 128 && kBits == 16 ? 3 : 4;
  static constexpr int kWide = 4 * kPerSm;
  // 4 bits: a warp's ring of steps, each the rows of 32 keys: key codes, value codes, key scales, value scales
  static constexpr int kKeys = kBits == 4 ? 32 : kStepKeys, kStages = kNT == 2 ? 4 : 2;
  static constexpr int kCodeBytes = kKeys * kD / 2, kScaleBytes = kKeys * kD / kGroup * 4;
  static constexpr int kStageBytes = 2 * kCodeBytes + 2 * kScaleBytes;
  static constexpr int kMergeBytes = 8 * kNT * kRow<kD> * 4;   // a warp's results (in its ring, where it has one)
  static constexpr int kWarpBytes = kBits == 4 ? kStages * kStageBytes : kMergeBytes;
  static_assert(kWarpBytes >= kMergeBytes && kWarpBytes % 16 == 0, "results fit the ring");
};

// ---- 16 bits
template <typename T, int kD, int kNT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 4 ? AttendCfg<kD, kNT, 16>::kPerSm : 1) paged_attention_kernel(const AttendParams p) {
  using Cfg = AttendCfg<kD, kNT, 16>;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr float kLazy = 8.f;
  extern __shared__ __align__(16) float smem_f[];
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Unit u = unit_of<kStepKeys>(p, 8 * kNT);
  if (u.rows <= 0) return;   // (all blocks of the cluster do)

  uint4 qf[kNT][kD / 32];   // Q^T fragments: of row 8n + g, the bytes this thread also reads of a key row
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int i = 0; i < kD / 32; ++i)
      qf[n][i] = 8 * n + g < u.rows ? *(reinterpret_cast<const uint4*>(query_row<T>(p, u, 8 * n + g)) + 4 * i + t) : make_uint4(0, 0, 0, 0);
  RowState<kNT, kD / 16, false> st;
  st.clear(u, t);
  const int32_t* table = p.c.table + static_cast<int64_t>(u.b) * p.c.table_stride;
  const int begin = u.begin + warp, end = u.end;
  bool bad_page = false;

  auto base_of = [&](int i) { return u.list.at(i) * kStepKeys; };
  auto entry_of = [&](int i) { return __ldg(table + (base_of(min(i, end - 1)) >> p.c.shift)); };   // (used where i < end)
  uint4 kf[2][kD / 32];   // key rows g, g + 8
  uint4 vf[4][kD / 64];   // value rows 2t, 2t + 1, 2t + 8, 2t + 9
  const T* const kbase = reinterpret_cast<const T*>(p.c.k) + 8 * t;
  const T* const vbase = reinterpret_cast<const T*>(p.c.v) + 8 * g;
  auto load_k_at = [&](uint32_t at, int next) {
    const T* src = kbase + static_cast<uint64_t>(at) * kD;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < kD / 32; ++j) kf[r][j] = __ldg(reinterpret_cast<const uint4*>(src + r * next * kD) + 4 * j);
  };
  auto load_v_at = [&](uint32_t at, int d1, int d2, int d3) {
    const T* src = vbase + static_cast<uint64_t>(at) * kD;
    const int far[4] = {0, d1, d2, d3};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < kD / 64; ++j) vf[r][j] = __ldg(reinterpret_cast<const uint4*>(src + far[r] * kD) + 8 * j);
  };
  auto load_k = [&](int base, uint32_t row) {
    if (whole_step<kStepKeys>(u, base)) {
      load_k_at(row + g, 8);
    } else {
      const int at = place<kStepKeys>(u, base, g);
      load_k_at(row + at, place<kStepKeys>(u, base, g + 8) - at);
    }
  };
  auto load_v = [&](int base, uint32_t row) {
    if (whole_step<kStepKeys>(u, base)) {
      load_v_at(row + 2 * t, 1, 8, 9);
    } else {
      const int at = place<kStepKeys>(u, base, 2 * t);
      load_v_at(row + at, place<kStepKeys>(u, base, 2 * t + 1) - at, place<kStepKeys>(u, base, 2 * t + 8) - at, place<kStepKeys>(u, base, 2 * t + 9) - at);
    }
  };
  // the next step's keys are loaded as soon as this one's are in the scores, its values behind this one's products
  if (begin < end) {
    int base = base_of(begin);
    uint32_t row = page_row(p.c, u.hk, entry_of(begin), base, &bad_page);
    load_k(base, row);
    load_v(base, row);
    int entry = entry_of(begin + kWarps);
    for (int i = begin; i < end; i += kWarps) {
      const int next = min(i + kWarps, end - 1), next_base = base_of(next);
      row = page_row(p.c, u.hk, entry, next_base, &bad_page);
      entry = entry_of(next + kWarps);
      float xs[1][kNT][4];
      float (&x)[kNT][4] = xs[0];
#pragma unroll
      for (int n = 0; n < kNT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < kD / 32; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816<T>(x[n], word_of(kf[0][j], 2 * half), word_of(kf[1][j], 2 * half), word_of(kf[0][j], 2 * half + 1),
                        word_of(kf[1][j], 2 * half + 1), word_of(qf[n][j], 2 * half), word_of(qf[n][j], 2 * half + 1));
      load_k(next_base, row);
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = fmaf(x[n][e], p.scale_log2, st.shift[n][e & 1]);
      if (edge_step<kStepKeys>(u, p, base)) st.mask(x, p, base + g, base + g + 8);
      st.probabilities(xs, kLazy);
      uint32_t pb[kNT][2];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        pb[n][0] = transpose8x8(pack_t<T>(x[n][0], x[n][1]));   // keys 2t, 2t + 1 of row g
        pb[n][1] = transpose8x8(pack_t<T>(x[n][2], x[n][3]));   // keys 2t + 8, 2t + 9
      }
#pragma unroll
      for (int h = 0; h < kD / 64; ++h)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t a0 = __byte_perm(word_of(vf[0][h], q), word_of(vf[1][h], q), 0x5410);   // element d of keys 2t, 2t + 1
          const uint32_t a1 = __byte_perm(word_of(vf[0][h], q), word_of(vf[1][h], q), 0x7632);   // element d + 1
          const uint32_t a2 = __byte_perm(word_of(vf[2][h], q), word_of(vf[3][h], q), 0x5410);   // keys 2t + 8, 2t + 9
          const uint32_t a3 = __byte_perm(word_of(vf[2][h], q), word_of(vf[3][h], q), 0x7632);
#pragma unroll
          for (int n = 0; n < kNT; ++n) mma16816<T>(st.o[n][4 * h + q], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
      load_v(next_base, row);
      base = next_base;
    }
  }
  bool good = u.good;
  if (__any_sync(kFull, bad_page)) {
    if (lane == 0) report_bad_index(p.c.status, 7);
    good = false;
  }
  float* mine = smem_f + warp * (Cfg::kWarpBytes / 4);
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float ls = st.l[n][e];
      ls += __shfl_xor_sync(kFull, ls, 4);
      ls += __shfl_xor_sync(kFull, ls, 8);
      ls += __shfl_xor_sync(kFull, ls, 16);
      float* row = mine + (8 * n + 2 * t + e) * kRow<kD>;
#pragma unroll
      for (int j = 0; j < kD / 16; ++j)
        *reinterpret_cast<float2*>(row + 64 * (j >> 2) + 8 * g + 2 * (j & 3)) = make_float2(st.o[n][j][e], st.o[n][j][2 + e]);
      if (g == 0) *reinterpret_cast<float2*>(row + kD) = good ? make_float2(st.m[n][e], ls) : make_float2(0.f, __uint_as_float(0x7fffffffu));
    }
  }
  merge<T, kD, kNT, kWarps>(p, u, smem_f, Cfg::kWarpBytes / 4);
}

// ---- 4 bits.  A step is 32 keys, 5 KB at D = 128, whose halves each lie together in four pieces: eight lanes of a warp fetch them
// with bulk copies into a ring of the warp's own, and the products read their fragments from there.
// (Fragments straight from global memory take 14 loads and their addresses for 16 keys, with a step or two in flight.)
// Shared memory would meet itself four times in a value row's bank if thread t took rows 2t and 2t + 1: slot s of a half is key
// (s / 2) + 4 (s % 2) of its eight instead, so that t takes rows t, t + 4, t + 8, t + 12.
template <typename T, int kD, int kNT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 4 ? AttendCfg<kD, kNT, 4>::kPerSm : 1) paged_attention_4bit_kernel(const AttendParams p) {
  using Cfg = AttendCfg<kD, kNT, 4>;
  constexpr int kGroups = kD / kGroup, kStages = Cfg::kStages, kKeys = Cfg::kKeys;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr float kLazy = std::is_same<T, __half>::value ? 2.f : 8.f;
  extern __shared__ __align__(16) float smem_f[];
  __shared__ uint64_t bars[kWarps][kStages];
  __shared__ uint32_t abort_flag;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const Unit u = unit_of<kKeys>(p, 8 * kNT);
  if (u.rows <= 0) return;   // (all blocks of the cluster do)
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < kStages; ++i) mbar_init(&bars[w][i], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  uint8_t* const ring = reinterpret_cast<uint8_t*>(smem_f) + warp * Cfg::kWarpBytes;
  const int32_t* table = p.c.table + static_cast<int64_t>(u.b) * p.c.table_stride;
  const int begin = u.begin + warp, end = u.end;
  bool bad_page = false;
  auto base_of = [&](int i) { return u.list.at(i) * kKeys; };
  // Step i into a slot of the ring: lane l < 8 fetches piece l % 4 of half l / 4, if a row sees a key of that half (the page of one
  // that none does may not be the sequence's any more).
  const int my_half = lane >> 2 & 1;
  const bool scales = lane & 1;
  const uint8_t* const piece_src = static_cast<const uint8_t*>(lane & 2 ? (scales ? p.c.v_scales : p.c.v) : (scales ? p.c.k_scales : p.c.k));
  const uint32_t piece_row = scales ? kGroups * 4 : kD / 2, piece_bytes = piece_row * kStepKeys;
  uint8_t* const piece_dst = ring + (scales ? 2 * Cfg::kCodeBytes : 0) + (lane & 2 ? 2 * static_cast<int>(piece_bytes) : 0) + my_half * piece_bytes;
  auto half_seen = [&](int from) {
    return from <= u.p_last && !(from >= u.hidden_from && min(from + kStepKeys - 1, u.p_last) < u.hidden_to);
  };
  auto entry_of = [&](int i) {   // (of a step there is; a half that nobody sees takes the other's)
    const int base = base_of(i), from = base + kStepKeys * my_half;
    return __ldg(table + ((half_seen(from) ? from : base + kStepKeys * (1 - my_half)) >> p.c.shift));
  };
  auto fetch = [&](int i, int entry, int slot) {
    const int from = base_of(i) + kStepKeys * my_half;
    const bool seen = half_seen(from);
    const uint32_t row = page_row(p.c, u.hk, entry, from, &bad_page);
    const unsigned halves = __ballot_sync(kFull, seen);   // bits 0 and 4
    uint64_t* bar = &bars[warp][slot];
    if (lane == 0) mbar_arrive_expect_tx(bar, Cfg::kStageBytes / 2 * ((halves & 1u) + (halves >> 4 & 1u)));
    __syncwarp();
    if (lane < 8 && seen) bulk_load_1d(piece_dst + slot * Cfg::kStageBytes, piece_src + static_cast<uint64_t>(row) * piece_row, piece_bytes, bar);
  };
#pragma unroll
  for (int j = 0; j < kStages; ++j) {
    if (begin + j * kWarps < end) fetch(begin + j * kWarps, entry_of(begin + j * kWarps), j);
  }
  int entry = begin + kStages * kWarps < end ? entry_of(begin + kStages * kWarps) : 0;

  // Q^T fragments of row 8n + g, as fp16 times a power of two, and the sums of its groups in three parts
  uint32_t qf[kNT][kD / 8], qs[kNT][2];   // qs: thread t has the t-th parts of groups (0, 1) and (2, 3)
  float scale[kNT][2];                    // of the scores of rows 2t and 2t + 1, to the log2 domain
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    float q[kD / 4], top = 0.f;   // this thread's eight of every 32 elements
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (8 * n + g < u.rows) x = *reinterpret_cast<const uint4*>(query_row<T>(p, u, 8 * n + g) + 32 * i + 8 * t);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        q[8 * i + j] = j & 1 ? hi_f32(word_of(x, j >> 1), T()) : lo_f32(word_of(x, j >> 1), T());
        top = fmaxf(top, fabsf(q[8 * i + j]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
    const uint32_t ex = min(__float_as_uint(top) >> 23, 253u);
    const float down = __uint_as_float((254u - ex) << 23), up = __uint_as_float(ex << 23);
    float part[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // pairs of elements four apart, as the codes of a word come
        const uint32_t w = pack2<false>(q[8 * i + j] * down, q[8 * i + j + 4] * down);
        qf[n][4 * i + j] = w;
        sum += lo_f32(w, __half()) + hi_f32(w, __half());
      }
      sum += __shfl_xor_sync(kFull, sum, 1);
      sum += __shfl_xor_sync(kFull, sum, 2);   // of row 8n + g, in every thread of the quad
#pragma unroll
      for (int v = 0; v < 3; ++v) {
        const float r = round_t<T>(sum);
        part[i] = t == v ? r : v == 0 ? 0.f : part[i];
        sum -= r;
      }
    }
    qs[n][0] = pack_t<T>(part[0], part[1]);
    qs[n][1] = kGroups > 2 ? pack_t<T>(part[kGroups - 2], part[kGroups - 1]) : 0;
    scale[n][0] = p.scale_log2 * __shfl_sync(kFull, up, 8 * t);
    scale[n][1] = p.scale_log2 * __shfl_sync(kFull, up, 8 * t + 4);
  }
  RowState<kNT, kD / 16, true> st;
  st.clear(u, t);
  const uint32_t one_v = std::is_same<T, __half>::value ? p.one_f16 : p.one_bf16;
  const uint32_t z_halves = (g / kGroups) & 1 ? 0x7632 : 0x5410;
  const int k_first = (g >> 1) + 4 * (g & 1);   // key of slot g

  auto step = [&](const uint8_t* stage, int base, auto simple) {
    constexpr bool kSimple = decltype(simple)::value;   // every row sees every key
    int kr[2][2], vr[2][4];                             // [half]: rows of the stage
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < 2; ++r) kr[h][r] = 16 * h + k_first + 8 * r;
#pragma unroll
      for (int r = 0; r < 4; ++r) vr[h][r] = 16 * h + t + 4 * r;
      if (!kSimple) {
#pragma unroll
        for (int r = 0; r < 2; ++r) kr[h][r] = place<kKeys>(u, base, kr[h][r]);
#pragma unroll
        for (int r = 0; r < 4; ++r) vr[h][r] = place<kKeys>(u, base, vr[h][r]);
      }
    }
    const uint8_t* const kc = stage + t * (kD / 8);
    const uint8_t* const vc = stage + Cfg::kCodeBytes + g * (kD / 16);
    const uint8_t* const ksc = stage + 2 * Cfg::kCodeBytes;
    const uint8_t* const vsc = ksc + Cfg::kScaleBytes;
    auto words = [&](const uint8_t* src, auto& w) {   // 4, 8 or 16 bytes
      constexpr int n = sizeof(w) / 4;
      if constexpr (n == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(src);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      } else if constexpr (n == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(src);
        w[0] = x.x; w[1] = x.y;
      } else {
        w[0] = *reinterpret_cast<const uint32_t*>(src);
      }
    };
    float x[2][kNT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < kNT; ++n) x[h][n][0] = x[h][n][1] = x[h][n][2] = x[h][n][3] = 0.f;
      uint32_t ks[2][kGroups], k[2][kGroups];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        words(ksc + kr[h][r] * (kGroups * 4), ks[r]);
        words(kc + kr[h][r] * (kD / 2), k[r]);
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n)   // keys by groups: minima times sums
        mma16816<T>(x[h][n], __byte_perm(ks[0][0], ks[0][1], 0x7632), __byte_perm(ks[1][0], ks[1][1], 0x7632),
                    kGroups > 2 ? __byte_perm(ks[0][kGroups - 2], ks[0][kGroups - 1], 0x7632) : 0u,
                    kGroups > 2 ? __byte_perm(ks[1][kGroups - 2], ks[1][kGroups - 1], 0x7632) : 0u, qs[n][0], qs[n][1]);
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        float acc[kNT][4];
#pragma unroll
        for (int n = 0; n < kNT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        uint32_t a[4], c[4];
        codes_of<__half>(k[0][G], 0.f, p.one_f16, a);
        codes_of<__half>(k[1][G], 0.f, p.one_f16, c);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816<__half>(acc[n], a[2 * j], c[2 * j], a[2 * j + 1], c[2 * j + 1], qf[n][4 * G + 2 * j], qf[n][4 * G + 2 * j + 1]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float s = lo_f32(ks[r][G], T());
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[h][n][2 * r + e] = fmaf(s, acc[n][2 * r + e], x[h][n][2 * r + e]);
        }
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h][n][e] = fmaf(x[h][n][e], scale[n][e & 1], st.shift[n][e & 1]);
      if (!kSimple) st.mask(x[h], p, base + 16 * h + k_first, base + 16 * h + k_first + 8);
    }
    st.probabilities(x, kLazy);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t vs[2][kGroups], v[4][kD / 64];
#pragma unroll
      for (int r = 0; r < 2; ++r) words(vsc + kr[h][r] * (kGroups * 4), vs[r]);
      {
        uint32_t zs[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          words(vc + vr[h][r] * (kD / 2), v[r]);
          zs[r] = *reinterpret_cast<const uint32_t*>(vsc + vr[h][r] * (kGroups * 4) + (g % kGroups) * 4);
        }
        const uint32_t a0 = __byte_perm(zs[0], zs[1], z_halves), a2 = __byte_perm(zs[2], zs[3], z_halves);
#pragma unroll
        for (int n = 0; n < kNT; ++n)
          mma16816<T>(st.z[n], a0, 0u, a2, 0u, transpose8x8(pack_t<T>(x[h][n][0], x[h][n][1])), transpose8x8(pack_t<T>(x[h][n][2], x[h][n][3])));
      }
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        uint32_t pb[kNT][2];
        const float vs0 = lo_f32(vs[0][G], T()), vs1 = lo_f32(vs[1][G], T());
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          pb[n][0] = transpose8x8(pack_t<T>(x[h][n][0] * vs0, x[h][n][1] * vs0));
          pb[n][1] = transpose8x8(pack_t<T>(x[h][n][2] * vs1, x[h][n][3] * vs1));
        }
        // elements 32 G + 4 g + 0..3 of the two pairs of keys
        uint32_t a[4], c[4];
        codes_of<T>(__byte_perm(v[0][G >> 1], v[1][G >> 1], G & 1 ? 0x7632 : 0x5410), 8.f, one_v, a);
        codes_of<T>(__byte_perm(v[2][G >> 1], v[3][G >> 1], G & 1 ? 0x7632 : 0x5410), 8.f, one_v, c);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int n = 0; n < kNT; ++n) mma16816<T>(st.o[n][2 * G + j], a[2 * j], a[2 * j + 1], c[2 * j], c[2 * j + 1], pb[n][0], pb[n][1]);
      }
    }
  };

  bool good = u.good;
  int slot = 0;
  uint32_t phase = 0;
  for (int i = begin; i < end; i += kWarps) {
    if (!mbar_wait_warp(&bars[warp][slot], phase, &abort_flag, p.c.status, 0xc00, p.wait_budget)) {
      good = false;
      break;
    }
    const uint8_t* stage = ring + slot * Cfg::kStageBytes;
    const int base = base_of(i);
    if (edge_step<kKeys>(u, p, base)) step(stage, base, std::false_type());
    else step(stage, base, std::true_type());
    __syncwarp();   // every lane is done with the slot
    const int later = i + kStages * kWarps;
    if (later < end) {
      fetch(later, entry, slot);
      if (later + kWarps < end) entry = entry_of(later + kWarps);
    }
    if (++slot == kStages) { slot = 0; phase ^= 1; }
  }
  settle_if_aborted(&abort_flag);
  if (__any_sync(kFull, bad_page)) {
    if (lane == 0) report_bad_index(p.c.status, 7);
    good = false;
  }
  // (every copy of the warp has arrived: its results take the ring's place)
  float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float ls = st.l[n][e];
      ls += __shfl_xor_sync(kFull, ls, 4);
      ls += __shfl_xor_sync(kFull, ls, 8);
      ls += __shfl_xor_sync(kFull, ls, 16);
      float* row = mine + (8 * n + 2 * t + e) * kRow<kD>;
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        const float zs = fmaf(8.f, __shfl_sync(kFull, st.z[n][e], 4 * G + t), __shfl_sync(kFull, st.z[n][e], 4 * (kGroups + G) + t));
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float2*>(row + 32 * G + 4 * g + 2 * j) = make_float2(st.o[n][2 * G + j][e] + zs, st.o[n][2 * G + j][2 + e] + zs);
      }
      if (g == 0) *reinterpret_cast<float2*>(row + kD) = good ? make_float2(st.m[n][e], ls) : make_float2(0.f, __uint_as_float(0x7fffffffu));
    }
  }
  merge<T, kD, kNT, kWarps>(p, u, smem_f, Cfg::kWarpBytes / 4);
}

// rows of a unit, and units, of a call
int64_t tile_of(int64_t heads_q, int64_t heads_kv, int64_t S) { return heads_q / heads_kv * S <= 8 ? 8 : 16; }
int64_t units_of(int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t S) {
  const int64_t tile = tile_of(heads_q, heads_kv, S);
  return batch * heads_kv * ((heads_q / heads_kv * S + tile - 1) / tile);
}

// Several clusters share a unit where there are few units and many keys: one cluster has 16 SMs.  B200, us of the kernels, caches cold, one
// token, D = 128, one cluster (no workspace) / teams: B1 Hq8 Hkv1, 16384 keys 15.4 / 11.8, 65536 40.5 / 20.2, 131072 73 / 23; B1 Hq32 Hkv4,
// 131072 73 / 51; B2 Hq32 Hkv8, 131072 196 / 160, with 4 bits 143 / 100; 8192 keys and fewer never gain.  The join (a kernel of its own) is
// entered dearer than it is, 6 us for about 3: where that decides, the model is no better than its 5 % (B7 Hkv1, 131072 keys, 16 bits 77 /
// 86; B1 Hq8 Hkv8 D64, 23508 keys, 16 bits 16.7 / 17.4: the two that lose among 48).
constexpr int64_t kTeamKeys = B200FA_PAGED_TEAM_KEYS, kTeamUnits = 128;
constexpr double kJoinCost = 6.0;   // us

// How a unit's keys are shared: `teams` clusters of `peers` blocks, of four warps each or, `wide`, of as many as an SM takes.
struct Shares {
  int peers, teams;
  bool wide;
};
// The cheapest by this model, in us and keys of a unit: a block alone works through `alone` (`alone_wide`) keys a us, all of them
// together through `total`, and the two add up as cubes; `fits` clusters run at once (they do not cross a GPC: asked of the device),
// and a last wave that is not full costs nearly as much as a full one; a peer costs 0.39 us, a wide block 1.9.  Fitted on 7037 random
// calls (1-1024 units, 64-65536 keys, spread by up to 90 %, which the host does not know, windows among them) with every share of up to
// 16 forced: the choice takes 4.7 % more time than each call's best (99 in 100: at most 26 %); as many blocks as fit at once, 21 %.
// B200, us, four-warp blocks 1 / 4 / 8 / 16 and 12-warp blocks 1 / 4 / 8 / 16: B8 Hq32 Hkv8 Sk32768 spread 60 % D128 16 bits 468 / 153 / 139 /
// 149, 267 / 134 / 154 / 202; B1 Hq8 Hkv1 Sk65536 888 / 228 / 120 / 66, 527 / 140 / 76 / 44.
Shares choose_shares(int64_t units, int64_t keys, int D, int bits, int row_tile, int max_teams, const int* fits, const int* fits_wide) {
  static constexpr float kRates[2][2][2][3] = {   // [D = 128][16 bits][two tiles of rows]: alone, alone_wide, total
      {{{92, 240, 33000}, {99, 56, 18000}}, {{130, 280, 63000}, {100, 200, 17000}}},
      {{{56, 120, 11000}, {57, 91, 5700}}, {{75, 130, 15000}, {90, 33, 12000}}}};
  const float* rate = kRates[D == 128][bits == 16][row_tile == 2];
  Shares best = {1, 1, false};
  double least = -1.0;
  for (int wide = 0; wide < 2; ++wide) {
    for (int peers = 1; peers <= kMaxPeers; ++peers) {
      const int fit = (wide ? fits_wide : fits)[peers];
      if (fit < 1) continue;
      const double all = static_cast<double>(units) * keys / rate[2];
      for (int teams = 1; teams <= (peers % 8 == 0 ? max_teams : 1); ++teams) {
        const double x = static_cast<double>(units) * teams / fit, waves = 0.89 * std::ceil(x) + 0.11 * x;
        const double chain = waves * keys / (peers * teams) / rate[wide];
        const double fixed = (wide ? 1.9 : 0.0) + (peers > 1 ? 0.39 * peers : 0.0) + (teams > 1 ? kJoinCost : 0.0);
        if (least >= 0.0 && fixed + std::max(all, chain) >= least) continue;   // (most; the root takes a short call's host longer than the rest)
        const double cost = fixed + std::cbrt(all * all * all + chain * chain * chain);
        if (least < 0.0 || cost < least) {
          least = cost;
          best = Shares{peers, teams, wide != 0};
        }
      }
    }
  }
  return best;
}

template <typename T, int kD, int kNT, int kBits, int kWarps>
constexpr auto attention_kernel() {
  if constexpr (kBits == 4) return &paged_attention_4bit_kernel<T, kD, kNT, kWarps>;
  else return &paged_attention_kernel<T, kD, kNT, kWarps>;
}

template <int kD, int kNT, int kBits, int kWarps>
void config_of(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, dim3 grid, int peers, cudaStream_t stream) {
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = peers;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  *cfg = cudaLaunchConfig_t{};
  cfg->gridDim = grid;
  cfg->blockDim = dim3(kWarps * 32);
  cfg->dynamicSmemBytes = kWarps * AttendCfg<kD, kNT, kBits>::kWarpBytes;
  cfg->stream = stream;
  cfg->attrs = attr;
  cfg->numAttrs = peers > 1 ? 1 : 0;
}

// Clusters of 1 .. 16 blocks of a kernel that the current device runs at once; the kernel is made ready for them.  Once per device.
template <typename T, int kD, int kNT, int kBits, int kWarps>
cudaError_t clusters_that_fit(const int** fits) {
  constexpr auto kern = attention_kernel<T, kD, kNT, kBits, kWarps>();
  static std::once_flag once[64];
  static cudaError_t result[64];
  static int count[64][kMaxPeers + 1];
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (r == cudaSuccess) r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kWarps * AttendCfg<kD, kNT, kBits>::kWarpBytes);
    for (int peers = 1; peers <= kMaxPeers && r == cudaSuccess; ++peers) {
      config_of<kD, kNT, kBits, kWarps>(&cfg, &attr, dim3(peers), peers, nullptr);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&count[dev][peers], kern, &cfg) != cudaSuccess) {   // then never of this size
        (void)cudaGetLastError();
        count[dev][peers] = 0;
      }
    }
    result[dev] = r;
  });
  *fits = count[dev];
  return result[dev];
}

// How a call's keys are shared, with `part_bytes` of workspace; 0 bytes are one cluster's share too.
template <typename T, int kD, int kNT, int kBits>
cudaError_t shares_of(const AttendParams& p, int64_t keys, size_t part_bytes, Shares* s) {
  const int *fits = nullptr, *fits_wide = nullptr;
  cudaError_t e = clusters_that_fit<T, kD, kNT, kBits, 4>(&fits);
  if (e == cudaSuccess) e = clusters_that_fit<T, kD, kNT, kBits, AttendCfg<kD, kNT, kBits>::kWide>(&fits_wide);
  if (e != cudaSuccess) return e;
  const int64_t room = part_bytes / paged_part_bytes(p.c.B, p.Hq, p.c.Hkv, p.S, kD);
  const int max_teams = std::max<int64_t>(1, std::min<int64_t>(room, paged_teams(p.c.B, p.Hq, p.c.Hkv, p.S, keys)));
  *s = choose_shares(units_of(p.c.B, p.Hq, p.c.Hkv, p.S), keys, kD, kBits, kNT, max_teams, fits, fits_wide);
  return e;
}

template <typename T, int kD, int kNT, int kBits>
cudaError_t launch_attend(AttendParams p, int64_t keys, size_t part_bytes, cudaStream_t stream, int* launches) {
  constexpr int kWide = AttendCfg<kD, kNT, kBits>::kWide;
  Shares s;
  cudaError_t e = shares_of<T, kD, kNT, kBits>(p, keys, part_bytes, &s);
  if (e != cudaSuccess) return e;
  p.group = p.Hq / p.c.Hkv;
  const int row_tiles = (p.group * p.S + 8 * kNT - 1) / (8 * kNT);
  p.one_f16 = kOneF16;
  p.one_bf16 = kOneBf16;
  p.peers = s.peers;
  p.teams = s.teams;
  const dim3 grid(s.peers * s.teams * row_tiles, p.c.Hkv, p.c.B);
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  if (s.wide) {
    config_of<kD, kNT, kBits, kWide>(&cfg, &attr, grid, s.peers, stream);
    e = cudaLaunchKernelEx(&cfg, attention_kernel<T, kD, kNT, kBits, kWide>(), p);
  } else {
    config_of<kD, kNT, kBits, 4>(&cfg, &attr, grid, s.peers, stream);
    e = cudaLaunchKernelEx(&cfg, attention_kernel<T, kD, kNT, kBits, 4>(), p);
  }
  if (e != cudaSuccess) return e;
  *launches += 1;
  if (s.teams == 1) return e;
  p.peers = p.teams = 1;
  paged_join_kernel<T, kD, 8 * kNT><<<dim3(row_tiles, p.c.Hkv, p.c.B), kJoinThreads, 0, stream>>>(p, s.teams);
  *launches += 1;
  return cudaGetLastError();
}

template <typename T, int kD, int kBits>
cudaError_t launch_attend_rows(const AttendParams& p, int64_t keys, size_t part_bytes, cudaStream_t stream, int* launches) {
  return tile_of(p.Hq, p.c.Hkv, p.S) == 8 ? launch_attend<T, kD, 1, kBits>(p, keys, part_bytes, stream, launches)
                                          : launch_attend<T, kD, 2, kBits>(p, keys, part_bytes, stream, launches);
}

// calls f with a value of the cache's type, its head dimension and its bits as constants
template <typename F>
cudaError_t with_cache(const PagedCache& c, int dtype, F f) {
  using std::integral_constant;
  auto with_bits = [&](auto type, auto d) {
    return c.bits == 4 ? f(type, d, integral_constant<int, 4>()) : f(type, d, integral_constant<int, 16>());
  };
  auto with_d = [&](auto type) {
    return c.D == 64 ? with_bits(type, integral_constant<int, 64>()) : with_bits(type, integral_constant<int, 128>());
  };
  return dtype == kBF16 ? with_d(__nv_bfloat16()) : with_d(__half());
}

}  // namespace

cudaError_t launch_paged_append(const AppendParams& p, int dtype, cudaStream_t stream, int* launches) {
  const cudaError_t e = with_cache(p.c, dtype, [&](auto type, auto d, auto bits) {
    using T = decltype(type);
    constexpr int kChunk = AppendCfg<T, d>::kChunk;
    const int64_t warps = static_cast<int64_t>(p.c.B) * p.S * ((p.Hq + kChunk - 1) / kChunk + 2 * ((p.c.Hkv + kChunk - 1) / kChunk));
    const unsigned blocks = static_cast<unsigned>((warps + 3) / 4);
    const auto kernel = p.clear ? (p.interleaved ? &paged_append_kernel<T, d, bits, true, true> : &paged_append_kernel<T, d, bits, false, true>)
                                : (p.interleaved ? &paged_append_kernel<T, d, bits, true, false> : &paged_append_kernel<T, d, bits, false, false>);
    kernel<<<blocks, 128, 0, stream>>>(p);
    return cudaGetLastError();
  });
  if (e == cudaSuccess && launches) *launches += 1;
  return e;
}

cudaError_t launch_paged_gather(const GatherParams& p, int dtype, cudaStream_t stream, int* launches) {
  const cudaError_t e = with_cache(p.c, dtype, [&](auto type, auto d, auto bits) {
    const int64_t threads = static_cast<int64_t>(p.c.B) * p.c.Hkv * p.S * (d / 8);
    paged_gather_kernel<decltype(type), d, bits><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(p);
    return cudaGetLastError();
  });
  if (e == cudaSuccess && launches) *launches += 1;
  return e;
}

cudaError_t launch_paged_attention(const AttendParams& p, int dtype, int64_t keys, size_t part_bytes, cudaStream_t stream, int* launches) {
  return with_cache(p.c, dtype, [&](auto type, auto d, auto bits) {
    return launch_attend_rows<decltype(type), d, bits>(p, keys, part_bytes, stream, launches);
  });
}

cudaError_t paged_shares(const AttendParams& p, int dtype, int64_t keys, size_t part_bytes, int* peers, int* teams, int* warps) {
  return with_cache(p.c, dtype, [&](auto type, auto d, auto bits) {
    using T = decltype(type);
    Shares s;
    const bool one_tile = tile_of(p.Hq, p.c.Hkv, p.S) == 8;
    const cudaError_t e = one_tile ? shares_of<T, d, 1, bits>(p, keys, part_bytes, &s) : shares_of<T, d, 2, bits>(p, keys, part_bytes, &s);
    if (e != cudaSuccess) return e;
    *peers = s.peers;
    *teams = s.teams;
    *warps = !s.wide ? 4 : one_tile ? AttendCfg<d, 1, bits>::kWide : AttendCfg<d, 2, bits>::kWide;
    return e;
  });
}

size_t paged_part_bytes(int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t S, int64_t D) {
  return sizeof(float) * units_of(batch, heads_q, heads_kv, S) * tile_of(heads_q, heads_kv, S) * (D + 4);
}

int paged_teams(int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t S, int64_t keys) {
  return keys < kTeamKeys ? 1 : static_cast<int>(std::min<int64_t>(kMaxTeams, std::max<int64_t>(1, kTeamUnits / units_of(batch, heads_q, heads_kv, S))));
}

}  // namespace b200fa
