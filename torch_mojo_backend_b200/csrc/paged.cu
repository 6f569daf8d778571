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
#include <atomic>
#include <mutex>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

// ------------------------------------------------------------------------------------------
// Append.  D / 8 lanes take a row (16 bytes each): one head's query, key or value of one token.  With (a, b) a pair of
// elements that turn together (i and i + R / 2, or 2 i and 2 i + 1, of the first R) and (c, s) its position's cos and sin,
// a' = a c - b s, b' = b c + a s: every product and sum rounded to fp32 on its own (no FMA), then to the type, so that the
// results are those of the formula in fp32 whatever computes it.  Copy-bound: each element is read and written once.
// A row of 4 bits: scale = (max - min) / 15 rounded to the type, code = round((x - min) / scale), of the elements as rounded to
// the type.  Where an element of a group is not finite the scale is NaN, and so is the group.
// ------------------------------------------------------------------------------------------
template <typename T, int kD, int kBits, bool kInterleaved>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  constexpr int kLanes = kD / 8;
  constexpr unsigned kFull = 0xffffffffu;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int li = static_cast<int>(threadIdx.x) % kLanes;
  const int64_t row = idx / kLanes;   // (token, head): heads of q, then of k, then of v
  const int heads = p.Hq + 2 * p.c.Hkv;
  const int64_t tokens = static_cast<int64_t>(p.c.B) * p.S;
  const bool inside = row < tokens * heads;
  const int64_t token = inside ? row / heads : 0;
  int h = inside ? static_cast<int>(row - token * heads) : 0;
  const int b = static_cast<int>(token / p.S), s = static_cast<int>(token - static_cast<int64_t>(b) * p.S);
  Sequence seq;
  const bool good = sequence_of(p.c, b, p.S, &seq);
  const int pos = seq.len - seq.n + s;
  bool write = inside && good && s < seq.n && pos >= 0;
  const bool angles = p.rotary == 0 || pos < p.positions;
  if (inside && (!good || (write && !angles))) {
    if (li == 0) report_bad_index(p.c.status, good ? 2 : 1);
    write = false;
  }
  const int what = h < p.Hq ? 0 : h < p.Hq + p.c.Hkv ? 1 : 2;   // q, k, v
  if (what == 1) h -= p.Hq;
  if (what == 2) h -= p.Hq + p.c.Hkv;
  int64_t at = 0;   // the row in the pages
  if (write && what != 0) {
    const int page = __ldg(p.c.table + static_cast<int64_t>(b) * p.c.table_stride + (pos >> p.c.shift));
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.pages)) {
      if (li == 0) report_bad_index(p.c.status, 3);
      write = false;
    } else {
      at = ((static_cast<int64_t>(page) * p.c.Hkv + h) << p.c.shift) + (pos & ((1 << p.c.shift) - 1));
    }
  }
  const View4& src = what == 0 ? p.q : what == 1 ? p.k : p.v;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (write)
    x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(src.ptr) + static_cast<int64_t>(b) * src.sb + static_cast<int64_t>(h) * src.sh +
                                        static_cast<int64_t>(s) * src.ss + li * 8);
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if (p.rotary) {
    const int e0 = li * 8, half = p.rotary / 2;
    const bool turn = write && what != 2 && e0 < p.rotary;
    if constexpr (kInterleaved) {
      if (turn) {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos + static_cast<int64_t>(pos) * half + e0 / 2));
        const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin + static_cast<int64_t>(pos) * half + e0 / 2));
        const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = lo_f32(w[i], T()), d = hi_f32(w[i], T());
          w[i] = pack_t<T>(__fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(d, sn[i])), __fadd_rn(__fmul_rn(d, cs[i]), __fmul_rn(a, sn[i])));
        }
      }
    } else {
      // the other elements of the pairs are half / 8 lanes away
      const bool first = e0 < half;
      const int lane = threadIdx.x & 31;
      const int from = e0 < p.rotary ? (first ? lane + half / 8 : lane - half / 8) : lane;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(kFull, w[i], from);
      if (turn) {
        const int64_t angle = static_cast<int64_t>(pos) * half + (first ? e0 : e0 - half);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos + angle) + i);
          const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin + angle) + i);
          const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t mine = w[2 * i + (j >> 1)], other = o[2 * i + (j >> 1)];
            const float a = j & 1 ? hi_f32(mine, T()) : lo_f32(mine, T()), d = j & 1 ? hi_f32(other, T()) : lo_f32(other, T());
            const float ac = __fmul_rn(a, cs[j]), ds = __fmul_rn(d, sn[j]);
            y[j] = first ? __fsub_rn(ac, ds) : __fadd_rn(ac, ds);
          }
          w[2 * i] = pack_t<T>(y[0], y[1]);
          w[2 * i + 1] = pack_t<T>(y[2], y[3]);
        }
      }
    }
  }
  if (what == 0) {
    if (write)
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out.ptr) + static_cast<int64_t>(b) * p.q_out.sb + static_cast<int64_t>(h) * p.q_out.sh +
                                static_cast<int64_t>(s) * p.q_out.ss + li * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if constexpr (kBits == 16) {
    if (write && what != 0) {
      void* pages = what == 1 ? p.c.k : p.c.v;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(pages) + at * kD + li * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    // the four lanes of a group find its minimum and maximum
    float v[8], low = INFINITY, high = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = i & 1 ? hi_f32(w[i >> 1], T()) : lo_f32(w[i >> 1], T());
      odd |= !(fabsf(v[i]) <= 3.402823466e38f);
      low = fminf(low, v[i]);
      high = fmaxf(high, v[i]);
    }
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
      low = fminf(low, __shfl_xor_sync(kFull, low, off));
      high = fmaxf(high, __shfl_xor_sync(kFull, high, off));
    }
    const unsigned odd_lanes = __ballot_sync(kFull, odd);
    if (!write || what == 0) return;
    float scale = round_t<T>(__fdiv_rn(__fsub_rn(high, low), 15.f));
    if ((odd_lanes >> ((threadIdx.x & 31) & ~3)) & 15u) scale = __uint_as_float(0x7fffffffu);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = rintf(__fdiv_rn(__fsub_rn(v[i], low), scale));
      const int code = scale > 0.f ? static_cast<int>(fminf(fmaxf(q, 0.f), 15.f)) : 0;
      codes |= static_cast<uint32_t>(code) << (4 * i);
    }
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

// ------------------------------------------------------------------------------------------
// Reading back.  D / 8 lanes take a row of k and the same row of v; rows behind a sequence's last are zero.  Copy-bound.
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
// token); a cluster of blocks shares its keys and merges (max, sum, O) through distributed shared memory.  A warp takes 16 keys a
// step, all in one page: S^T = K Q^T and O^T += V^T P^T by mma.sync m16n8k16, keys and then head-dim elements the M dimension,
// rows the N dimension, operands from global memory to fragment registers directly.  HBM-bound by design: K and V are read
// once per unit.  Thread (g, t) = (lane / 4, lane % 4) owns keys g and g + 8 and rows 2t and 2t + 1 of each tile in the softmax.
//   * 16 bits: K as thread (g, t) reads 16 bytes at (4i + t) 16 of key rows g and g + 8 (any permutation of the contraction
//     index will do if Q has the same); V as it reads 16 bytes at 128 h + 16 g of rows 2t, 2t+1, 2t+8, 2t+9, whose registers a
//     byte permute turns into (key, key + 1) pairs.
//   * 4 bits: a code c goes into the mantissa of 1.0, which makes 1 + c / 16 exactly, two codes per instruction; the scales stay
//     out of the products.  S = sum over groups G of 16 ks_G (q_G . c_G / 16) + km_G sum(q_G): the accumulator of a group
//     starts at -sum(q_G), which takes the ones off.  O_G = sum over keys of (P vs_G) c + P vm_G: P vs_G is the B operand, rounded
//     to bf16 whatever the cache's type (fp16 has not the range for a probability times a small scale), the ones are taken off
//     the codes, exactly, and sum(P vm_G) is the same for the 32 elements of a group: one fp32 number per row and group.
// The row maximum moves only when a score exceeds it by 2^8 (a vote per step instead of six shuffles), so P is at most 256.
// Keys that no row of the unit sees are never read, not even into a product with zero: their places in a step re-read a key that is
// seen (pages behind a window may have been given to another sequence).
// ------------------------------------------------------------------------------------------
constexpr int kStepKeys = 16;
constexpr int kWarps = 4;
constexpr int kMaxPeers = 16;
constexpr float kLazy = 8.f;

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

// Codes j of both halves of a word, each as 1 + code / 16
template <typename T, int j>
__device__ __forceinline__ uint32_t codes_plus_one(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {   // 7 bits of mantissa: the code goes to bits 3..6
    constexpr int s = 4 * j - 3;
    return ((s < 0 ? w << -s : w >> (s < 0 ? 0 : s)) & 0x00780078u) | 0x3f803f80u;
  } else {                                                 // 10 bits: to bits 6..9
    constexpr int s = 4 * j - 6;
    return ((s < 0 ? w << (s < 0 ? -s : 0) : w >> (s < 0 ? 0 : s)) & 0x03c003c0u) | 0x3c003c00u;
  }
}
__device__ __forceinline__ uint32_t minus_one_bf16x2(uint32_t x) {
  const __nv_bfloat162 one = __floats2bfloat162_rn(1.f, 1.f);
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), one);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 16 keys in registers
template <int kD, int kBits>
struct Fragments;
template <int kD>
struct Fragments<kD, 16> {
  uint4 k[2][kD / 32];   // key rows g, g + 8
  uint4 v[4][kD / 64];   // key rows 2t, 2t + 1, 2t + 8, 2t + 9
};
template <int kD>
struct Fragments<kD, 4> {
  uint32_t k[2][kD / 32];    // codes of key rows g, g + 8
  uint32_t ks[2][kD / 32];   // (scale, minimum) of their groups
  uint32_t vs[2][kD / 32];   // ... of the value rows g, g + 8
  uint32_t v[4][kD / 64];    // codes of value rows 2t, 2t + 1, 2t + 8, 2t + 9
};
template <int kN>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t (&w)[kN]) {
  if constexpr (kN == 4) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (kN == 2) {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = __ldg(p);
  }
}

// The last step of a unit: every block has left its unnormalised O of row r at o + r * (kD + 2) and the row's (max, sum) at ml + r, and
// merges its share of (row, pair of elements) from its peers' shared memory.
template <typename T, int kD, int kRows>
__device__ __forceinline__ void merge_peers(const AttendParams& p, int b, int hk, int group, int row0, int rows, int peers, int rank, const float* o,
                                            const float2* ml) {
  const int tid = threadIdx.x;
  if (peers > 1) cluster_sync(); else __syncthreads();
  for (int idx = rank * kWarps * 32 + tid; idx < rows * (kD / 2); idx += peers * kWarps * 32) {
    const int r = idx / (kD / 2), d = idx % (kD / 2) * 2;
    const uint32_t a_ml = smem_u32(ml + r), a_o = smem_u32(o + r * (kD + 2) + d);
    float2 v[kMaxPeers], x[kMaxPeers];
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) {
      if (i < peers) {
        v[i] = peer_load_f32x2(a_ml, i);
        x[i] = peer_load_f32x2(a_o, i);
      }
    }
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) {
      if (i < peers) m = fmaxf(m, v[i].x);
    }
    const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) {
      if (i < peers) {
        const float w = exp2f(v[i].x - m_use);   // 0 for a peer that saw no key of the row
        l = fmaf(v[i].y, w, l);
        o0 = fmaf(x[i].x, w, o0);
        o1 = fmaf(x[i].y, w, o1);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;   // a row without a key is 0 with lse -inf; a NaN stays one
    const int row = row0 + r, s = row / group, h = hk * group + row - s * group;
    T* dst = reinterpret_cast<T*>(p.out.ptr) + static_cast<int64_t>(b) * p.out.sb + static_cast<int64_t>(h) * p.out.sh + static_cast<int64_t>(s) * p.out.ss + d;
    *reinterpret_cast<uint32_t*>(dst) = pack_t<T>(o0 * inv, o1 * inv);
    if (d == 0) p.lse[(static_cast<int64_t>(b) * p.Hq + h) * p.S + s] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
  }
  if (peers > 1) cluster_sync();   // no block leaves while a peer may still read its shared memory
}

template <typename T, int kD, int kNT, int kBits>
__global__ void __launch_bounds__(kWarps * 32, kNT == 1 ? 3 : 2) paged_attention_kernel(const AttendParams p) {
  constexpr int kRows = 8 * kNT;
  constexpr int kGroups = kD / kGroup;
  constexpr int kTiles = kD / 16;   // tiles of O^T
  constexpr unsigned kFull = 0xffffffffu;
  __shared__ __align__(16) float sMerge[kWarps][kRows][kD + 2];   // per warp and row: O, then max and sum
  __shared__ float2 sML[kRows];
  const int peers = gridDim.x, rank = blockIdx.x, b = blockIdx.z;
  const int row_tiles = p.row_tiles;
  const int hk = blockIdx.y / row_tiles, row0 = (blockIdx.y - hk * row_tiles) * kRows;
  const int group = p.Hq / p.c.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;

  Sequence seq;
  bool good = sequence_of(p.c, b, p.S, &seq);
  if (!good) {   // every row of the sequence is NaN
    if (tid == 0) report_bad_index(p.c.status, 6);
    seq.len = 0;
    seq.n = p.S;
  }
  const int rows = min(kRows, seq.n * group - row0);   // of this unit
  if (rows <= 0) return;                               // (all blocks of the cluster do)
  const int first_pos = seq.len - seq.n;               // position of the first new token; negative: it sees nothing
  const int p_first = first_pos + row0 / group, p_last = first_pos + (row0 + rows - 1) / group;
  KeyBlocks list = {0, 0, max(0, p_last + kStepKeys) / kStepKeys};   // steps of 16 keys
  int hidden_from = 0, hidden_to = 0;                                // keys between the sinks and the first row's window
  if (p.window) {
    list = window_blocks<kStepKeys>(p_first, p_last, seq.len, p.window, p.sinks);
    hidden_from = p.sinks;
    hidden_to = p_first - p.window + 1;
  }
  const int begin = static_cast<int>(static_cast<int64_t>(list.n) * rank / peers), end = static_cast<int>(static_cast<int64_t>(list.n) * (rank + 1) / peers);

  // Q^T fragments of row 8n + g, and (4 bits) the sums of its groups
  uint32_t qf[kNT][kD / 8];
  float qs[kNT][2][kBits == 4 ? kGroups : 1];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const int r = 8 * n + g;
#pragma unroll
    for (int i = 0; i < kD / 8; ++i) qf[n][i] = 0;
    if (r < rows) {
      const int s = (row0 + r) / group, h = hk * group + row0 + r - s * group;
      const T* qp = reinterpret_cast<const T*>(p.q.ptr) + static_cast<int64_t>(b) * p.q.sb + static_cast<int64_t>(h) * p.q.sh + static_cast<int64_t>(s) * p.q.ss;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {   // 32 elements: this thread's eight
        const uint4 x = *reinterpret_cast<const uint4*>(qp + 32 * i + 8 * t);
        if constexpr (kBits == 16) {
          qf[n][4 * i] = x.x; qf[n][4 * i + 1] = x.y; qf[n][4 * i + 2] = x.z; qf[n][4 * i + 3] = x.w;
        } else {   // pairs of elements four apart, as the codes of a word come
          qf[n][4 * i] = __byte_perm(x.x, x.z, 0x5410); qf[n][4 * i + 1] = __byte_perm(x.x, x.z, 0x7632);
          qf[n][4 * i + 2] = __byte_perm(x.y, x.w, 0x5410); qf[n][4 * i + 3] = __byte_perm(x.y, x.w, 0x7632);
        }
      }
    }
    if constexpr (kBits == 4) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += lo_f32(qf[n][4 * i + j], T()) + hi_f32(qf[n][4 * i + j], T());
        sum += __shfl_xor_sync(kFull, sum, 1);
        sum += __shfl_xor_sync(kFull, sum, 2);   // of row 8n + g, in every thread of the quad
        qs[n][0][i] = __shfl_sync(kFull, sum, 8 * t);       // row 2t
        qs[n][1][i] = __shfl_sync(kFull, sum, 8 * t + 4);   // row 2t + 1
      }
    }
  }
  int pos[kNT][2];   // positions of rows 2t and 2t + 1 of each tile
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos[n][e] = first_pos + (row0 + 8 * n + 2 * t + e) / group;   // (rows behind the last are not written)
  float m[kNT][2], shift[kNT][2], limit[kNT][2], l[kNT][2];   // shift: -max, 0 as long as there is none; limit: where it moves
  float o[kNT][kTiles][4];
  float z[kNT][2][kBits == 4 ? kGroups : 1];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[n][e] = limit[n][e] = -INFINITY;
      shift[n][e] = l[n][e] = 0.f;
#pragma unroll
      for (int i = 0; i < (kBits == 4 ? kGroups : 1); ++i) z[n][e][i] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < kTiles; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
  }
  const int32_t* table = p.c.table + static_cast<int64_t>(b) * p.c.table_stride;
  bool bad_page = false;

  auto base_of = [&](int i) { return list.at(i) * kStepKeys; };
  auto entry_of = [&](int i) { return __ldg(table + (base_of(min(i, end - 1)) >> p.c.shift)); };   // (used where i < end)
  // row of the pages that holds the step's first key
  auto row_of = [&](int i, int page) {
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.pages)) {
      bad_page = true;
      page = 0;
    }
    return ((static_cast<int64_t>(page) * p.c.Hkv + hk) << p.c.shift) + (base_of(i) & ((1 << p.c.shift) - 1));
  };
  // place in the step of the key that is read for key `k` of it
  auto place = [&](int base, int k) {
    int key = min(base + k, p_last);
    if (key >= hidden_from && key < hidden_to) key = hidden_to < base + kStepKeys ? hidden_to : hidden_from - 1;
    return key - base;
  };
  const float scale = kBits == 4 ? p.scale_log2 * 16.f : p.scale_log2;

  using Frag = Fragments<kD, kBits>;
  auto load_k = [&](Frag& f, int i, int64_t row) {
    const int base = base_of(i);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t at = row + place(base, g + 8 * r);
      if constexpr (kBits == 16) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.c.k) + at * kD) + t;
#pragma unroll
        for (int j = 0; j < kD / 32; ++j) f.k[r][j] = __ldg(src + 4 * j);
      } else {
        load_words<kGroups>(reinterpret_cast<const uint32_t*>(p.c.k) + at * (kD / 8) + t * kGroups, f.k[r]);
        load_words<kGroups>(reinterpret_cast<const uint32_t*>(p.c.k_scales) + at * kGroups, f.ks[r]);
      }
    }
  };
  auto load_v = [&](Frag& f, int i, int64_t row) {
    const int base = base_of(i);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t at = row + place(base, 2 * t + (r & 1) + 8 * (r >> 1));
      if constexpr (kBits == 16) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.c.v) + at * kD) + g;
#pragma unroll
        for (int j = 0; j < kD / 64; ++j) f.v[r][j] = __ldg(src + 8 * j);
      } else {
        load_words<kD / 64>(reinterpret_cast<const uint32_t*>(p.c.v) + at * (kD / 8) + g * (kD / 64), f.v[r]);
      }
    }
    if constexpr (kBits == 4) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        load_words<kGroups>(reinterpret_cast<const uint32_t*>(p.c.v_scales) + (row + place(base, g + 8 * r)) * kGroups, f.vs[r]);
    }
  };
  // scores of a step's keys, scaled to the log2 domain less the rows' maxima: x[n][0] (key g, row 2t) [1] (key g, row 2t + 1) [2], [3] key g + 8
  auto scores = [&](const Frag& f, int i, float (&x)[kNT][4]) {
#pragma unroll
    for (int n = 0; n < kNT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
    if constexpr (kBits == 16) {
#pragma unroll
      for (int j = 0; j < kD / 32; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816<T>(x[n], word_of(f.k[0][j], 2 * half), word_of(f.k[1][j], 2 * half), word_of(f.k[0][j], 2 * half + 1),
                        word_of(f.k[1][j], 2 * half + 1), qf[n][4 * j + 2 * half], qf[n][4 * j + 2 * half + 1]);
    } else {
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        float acc[kNT][4];
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          acc[n][0] = acc[n][2] = -qs[n][0][G];
          acc[n][1] = acc[n][3] = -qs[n][1][G];
        }
        {
          const uint32_t a0 = codes_plus_one<T, 0>(f.k[0][G]), a1 = codes_plus_one<T, 0>(f.k[1][G]);
          const uint32_t a2 = codes_plus_one<T, 1>(f.k[0][G]), a3 = codes_plus_one<T, 1>(f.k[1][G]);
#pragma unroll
          for (int n = 0; n < kNT; ++n) mma16816<T>(acc[n], a0, a1, a2, a3, qf[n][4 * G], qf[n][4 * G + 1]);
        }
        {
          const uint32_t a0 = codes_plus_one<T, 2>(f.k[0][G]), a1 = codes_plus_one<T, 2>(f.k[1][G]);
          const uint32_t a2 = codes_plus_one<T, 3>(f.k[0][G]), a3 = codes_plus_one<T, 3>(f.k[1][G]);
#pragma unroll
          for (int n = 0; n < kNT; ++n) mma16816<T>(acc[n], a0, a1, a2, a3, qf[n][4 * G + 2], qf[n][4 * G + 3]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float ks = lo_f32(f.ks[r][G], T()), km = hi_f32(f.ks[r][G], T()) * 0.0625f;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[n][2 * r + e] = fmaf(ks, acc[n][2 * r + e], fmaf(km, qs[n][e][G], x[n][2 * r + e]));
        }
      }
    }
    const int base = base_of(i);
    // (a step at an edge: of some row's causal range, or of the span that some row's window leaves out)
    const bool edge = base + kStepKeys - 1 > p_first || (p.window && base <= p_last - p.window && base + kStepKeys - 1 >= p.sinks);
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[n][e] = fmaf(x[n][e], scale, shift[n][e & 1]);
        if (edge) {
          const int key = base + g + 8 * (e >> 1), at = pos[n][e & 1];
          if (key > at || (p.window && key <= at - p.window && key >= p.sinks)) x[n][e] = -INFINITY;
        }
      }
  };
  // raises the maxima of the rows that have a score too far above theirs, and rescales what was summed
  auto raise = [&](float (&x)[kNT][4]) {
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(x[n][e], x[n][2 + e]);
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 4));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 8));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 16));   // relative to the standing maximum (to 0 without one)
        const bool none = m[n][e] == -INFINITY;
        if (top > (none ? -INFINITY : 0.f)) {
          const float corr = none ? 0.f : exp2f(-top);
          m[n][e] = none ? top : m[n][e] + top;
          shift[n][e] = -m[n][e];
          limit[n][e] = kLazy;
          x[n][e] -= top;
          x[n][2 + e] -= top;
          l[n][e] *= corr;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            o[n][j][e] *= corr;
            o[n][j][2 + e] *= corr;
          }
          if constexpr (kBits == 4) {
#pragma unroll
            for (int G = 0; G < kGroups; ++G) z[n][e][G] *= corr;
          }
        }
      }
  };
  auto probabilities = [&](float (&x)[kNT][4]) {
    bool far = false;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) far |= fmaxf(x[n][e], x[n][2 + e]) > limit[n][e];
    if (__any_sync(kFull, far)) raise(x);
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] = ex2_approx(x[n][e]);
      l[n][0] += x[n][0] + x[n][2];   // this thread's two keys; summed over g at the end
      l[n][1] += x[n][1] + x[n][3];
    }
  };
  auto add_values = [&](const Frag& f, const float (&x)[kNT][4]) {
    if constexpr (kBits == 16) {
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
          const uint32_t a0 = __byte_perm(word_of(f.v[0][h], q), word_of(f.v[1][h], q), 0x5410);   // element d of keys 2t, 2t + 1
          const uint32_t a1 = __byte_perm(word_of(f.v[0][h], q), word_of(f.v[1][h], q), 0x7632);   // element d + 1
          const uint32_t a2 = __byte_perm(word_of(f.v[2][h], q), word_of(f.v[3][h], q), 0x5410);   // keys 2t + 8, 2t + 9
          const uint32_t a3 = __byte_perm(word_of(f.v[2][h], q), word_of(f.v[3][h], q), 0x7632);
#pragma unroll
          for (int n = 0; n < kNT; ++n) mma16816<T>(o[n][4 * h + q], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
    } else {
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        uint32_t pb[kNT][2];
        const float vs0 = lo_f32(f.vs[0][G], T()), vm0 = hi_f32(f.vs[0][G], T());
        const float vs1 = lo_f32(f.vs[1][G], T()), vm1 = hi_f32(f.vs[1][G], T());
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          pb[n][0] = transpose8x8(pack2<true>(x[n][0] * vs0, x[n][1] * vs0));
          pb[n][1] = transpose8x8(pack2<true>(x[n][2] * vs1, x[n][3] * vs1));
          z[n][0][G] = fmaf(x[n][0], vm0, fmaf(x[n][2], vm1, z[n][0][G]));
          z[n][1][G] = fmaf(x[n][1], vm0, fmaf(x[n][3], vm1, z[n][1][G]));
        }
        // elements 32 G + 4 g + 0..3 of keys (2t, 2t + 1) and (2t + 8, 2t + 9)
        const uint32_t ya = __byte_perm(f.v[0][G >> 1], f.v[1][G >> 1], G & 1 ? 0x7632 : 0x5410);
        const uint32_t yb = __byte_perm(f.v[2][G >> 1], f.v[3][G >> 1], G & 1 ? 0x7632 : 0x5410);
        uint32_t a[4], c[4];
        a[0] = codes_plus_one<__nv_bfloat16, 0>(ya); a[1] = codes_plus_one<__nv_bfloat16, 1>(ya);
        a[2] = codes_plus_one<__nv_bfloat16, 2>(ya); a[3] = codes_plus_one<__nv_bfloat16, 3>(ya);
        c[0] = codes_plus_one<__nv_bfloat16, 0>(yb); c[1] = codes_plus_one<__nv_bfloat16, 1>(yb);
        c[2] = codes_plus_one<__nv_bfloat16, 2>(yb); c[3] = codes_plus_one<__nv_bfloat16, 3>(yb);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[j] = minus_one_bf16x2(a[j]);
          c[j] = minus_one_bf16x2(c[j]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816<__nv_bfloat16>(o[n][2 * G + j], a[2 * j], a[2 * j + 1], c[2 * j], c[2 * j + 1], pb[n][0], pb[n][1]);
      }
    }
  };

  int i = begin + warp;
  if constexpr (kBits == 16) {
    // the next step's keys are loaded as soon as this one's are in the scores, its values behind this one's products
    if (i < end) {
      Frag f;
      int64_t row = row_of(i, entry_of(i));
      load_k(f, i, row);
      load_v(f, i, row);
      int entry = entry_of(i + kWarps);
      for (; i < end; i += kWarps) {
        const int next = min(i + kWarps, end - 1);
        row = row_of(next, entry);
        entry = entry_of(next + kWarps);
        float x[kNT][4];
        scores(f, i, x);
        load_k(f, next, row);
        probabilities(x);
        add_values(f, x);
        load_v(f, next, row);
      }
    }
  } else {
    // two steps of codes in flight: a step's are a quarter of the bytes
    if (i < end) {
      Frag f[2];
      int64_t row = row_of(i, entry_of(i));
      load_k(f[0], i, row);
      load_v(f[0], i, row);
      const int second = min(i + kWarps, end - 1);
      row = row_of(second, entry_of(second));
      load_k(f[1], second, row);
      load_v(f[1], second, row);
      int entry = entry_of(i + 2 * kWarps);
      while (true) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int next = min(i + 2 * kWarps, end - 1);
          row = row_of(next, entry);
          entry = entry_of(i + 3 * kWarps);
          float x[kNT][4];
          scores(f[u], i, x);
          load_k(f[u], next, row);
          probabilities(x);
          add_values(f[u], x);
          load_v(f[u], next, row);
          i += kWarps;
          if (i >= end) break;
        }
        if (i >= end) break;
      }
    }
  }
  if (__any_sync(kFull, bad_page)) {
    if (lane == 0) report_bad_index(p.c.status, 7);
    good = false;
  }
  // this warp's results to shared memory
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float ls = l[n][e];
      ls += __shfl_xor_sync(kFull, ls, 4);
      ls += __shfl_xor_sync(kFull, ls, 8);
      ls += __shfl_xor_sync(kFull, ls, 16);
      const int r = 8 * n + 2 * t + e;
      if constexpr (kBits == 16) {
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const int d = 64 * (j >> 2) + 8 * g + 2 * (j & 3);
          sMerge[warp][r][d] = o[n][j][e];
          sMerge[warp][r][d + 1] = o[n][j][2 + e];
        }
      } else {
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          float zs = z[n][e][G];
          zs += __shfl_xor_sync(kFull, zs, 4);
          zs += __shfl_xor_sync(kFull, zs, 8);
          zs += __shfl_xor_sync(kFull, zs, 16);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int d = 32 * G + 4 * g + 2 * j;
            sMerge[warp][r][d] = fmaf(16.f, o[n][2 * G + j][e], zs);
            sMerge[warp][r][d + 1] = fmaf(16.f, o[n][2 * G + j][2 + e], zs);
          }
        }
      }
      if (g == 0) {
        sMerge[warp][r][kD] = good ? m[n][e] : 0.f;
        sMerge[warp][r][kD + 1] = good ? ls : __uint_as_float(0x7fffffffu);
      }
    }
  }
  __syncthreads();
  // merge the warps
  for (int idx = tid; idx < rows * kD; idx += kWarps * 32) {
    const int r = idx / kD, d = idx % kD;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sMerge[w][r][kD]);
    const float m_use = mm == -INFINITY ? 0.f : mm;
    float acc = 0.f, ls = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float weight = exp2f(sMerge[w][r][kD] - m_use);
      acc = fmaf(sMerge[w][r][d], weight, acc);
      ls = fmaf(sMerge[w][r][kD + 1], weight, ls);
    }
    sMerge[0][r][d] = acc;   // (this thread alone reads and writes column d of row r)
    if (d == 0) sML[r] = make_float2(mm, ls);
  }
  merge_peers<T, kD, kRows>(p, b, hk, group, row0, rows, peers, rank, &sMerge[0][0][0], sML);
}

// Blocks that share a unit: enough to fill the GPU, of at least four steps for each warp of theirs.
int choose_peers(int64_t units, int64_t keys, int per_sm) {
  const int64_t steps = (keys + kStepKeys - 1) / kStepKeys;
  int64_t peers = 148 * per_sm / std::max<int64_t>(units, 1);
  peers = std::min(peers, steps / (4 * kWarps));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(peers, kMaxPeers)));
}

template <typename T, int kD, int kNT, int kBits>
cudaError_t launch_attend(AttendParams p, int64_t keys, cudaStream_t stream) {
  auto kern = paged_attention_kernel<T, kD, kNT, kBits>;
  static std::once_flag once[64];
  static cudaError_t result[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
  if (result[dev] != cudaSuccess) return result[dev];
  const int rows = p.Hq / p.c.Hkv * p.S;
  p.row_tiles = (rows + 8 * kNT - 1) / (8 * kNT);
  const int peers = choose_peers(static_cast<int64_t>(p.c.B) * p.c.Hkv * p.row_tiles, keys, kNT == 1 ? 3 : 2);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = peers;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(peers, p.c.Hkv * p.row_tiles, p.c.B);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = peers > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, int kD, int kBits>
cudaError_t launch_attend_rows(const AttendParams& p, int64_t keys, cudaStream_t stream) {
  return p.Hq / p.c.Hkv * p.S <= 8 ? launch_attend<T, kD, 1, kBits>(p, keys, stream) : launch_attend<T, kD, 2, kBits>(p, keys, stream);
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
    const int64_t threads = static_cast<int64_t>(p.c.B) * p.S * (p.Hq + 2 * p.c.Hkv) * (d / 8);
    const unsigned blocks = static_cast<unsigned>((threads + 255) / 256);
    if (p.interleaved) paged_append_kernel<T, d, bits, true><<<blocks, 256, 0, stream>>>(p);
    else paged_append_kernel<T, d, bits, false><<<blocks, 256, 0, stream>>>(p);
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

cudaError_t launch_paged_attention(const AttendParams& p, int dtype, int64_t keys, cudaStream_t stream, int* launches) {
  const cudaError_t e = with_cache(p.c, dtype, [&](auto type, auto d, auto bits) {
    return launch_attend_rows<decltype(type), d, bits>(p, keys, stream);
  });
  if (e == cudaSuccess && launches) *launches += 1;
  return e;
}

}  // namespace b200fa
