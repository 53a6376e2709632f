// What the attentions of drafted trees share, over pages of 16-bit rows
// (tree_attention.hip) and of 4-bit rows (tree_attention_int4.hip): their
// arguments, how the work is cut into equal shares, the launch that joins the
// parts, and the checks of an entry point.
#pragma once

#include "iron_common.hpp"
#include "int4_rows.hpp"
#include "../../include/iron_hip.h"

#include <algorithm>
#include <type_traits>

namespace iron {
namespace {

struct TreeArgs {
  const uint16_t* q;        // (num_nodes, H, D)
  const uint16_t* k_new;    // (num_nodes, Hkv, D)
  const uint16_t* v_new;
  const uint16_t* k_pages;  // (num_pages, Hkv, page_size, D), or 4-bit rows in the place of D values
  const uint16_t* v_pages;
  const int* table;   // (num_seqs, max_pages)
  const int* lens;    // (num_seqs)
  const int* starts;  // (num_seqs + 1)
  const int* mask;    // (num_nodes, words)
  uint16_t* out;      // (num_nodes, H, D)
  float* part_o;      // workspace (2 x workgroups, R, D): sum(p v) of the parts of split tiles
  float2* part_ml;    // workspace (2 x workgroups, R): their maximum and sum(p)
  int* prefix;        // workspace (num_seqs + 1): units before each sequence; units of a workgroup
  int* owner;         // workspace (num_nodes): the sequence of each node that is one
  int H, Hkv, G, num_pages, page_shift, num_seqs, max_pages, num_nodes, max_nodes, words, workgroups;
  float scale_log2;
};

template <bool F16>
__device__ __forceinline__ float widen(uint16_t x) {
  if constexpr (F16) return static_cast<float>(__builtin_bit_cast(_Float16, x));
  return bf16_to_f32(x);
}
template <bool F16>
__device__ __forceinline__ uint16_t narrow(float x) {
  if constexpr (F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
  return f32_to_bf16(x);
}

typedef __bf16 ta_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 ta_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 ta_f16x2 __attribute__((ext_vector_type(2)));
typedef float ta_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned ta_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned ta_u32x4 __attribute__((ext_vector_type(4)));
typedef short ta_i16x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 64;      // keys of a block: 16 for each of the 4 waves
constexpr int kWideBlock = 32;  // of the kernel of many rows
constexpr int kStages = 4;      // blocks resident in a ring

// fp16 weights are taken 2^6 times as large (at most 2^14 then), so that small
// ones stay in fp16's normal range six powers of two longer.
template <bool F16>
constexpr float kLift = F16 ? 6.f : 0.f;

template <bool F16>
__device__ __forceinline__ ta_f32x4 mfma(ta_u32x4 a, ta_u32x4 b, ta_f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ta_f16x8, a), __builtin_bit_cast(ta_f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ta_bf16x8, a), __builtin_bit_cast(ta_bf16x8, b), c, 0, 0, 0);
}

// Four weights as 16-bit pairs hi + lo: {hi0, hi1, hi2, hi3, lo0, lo1, lo2, lo3}.
// A weight keeps ~16 bits (bf16) or ~21 (fp16) that way: rounded to one 16-bit
// value it would add an error of the size of the output's own rounding.
template <bool F16>
__device__ __forceinline__ ta_u32x4 split4(const float (&p)[4]) {
  ta_u32x4 r;
  if constexpr (F16) {  // both parts truncate: what the first leaves off is never negative
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto hi = __builtin_amdgcn_cvt_pkrtz(p[2 * i], p[2 * i + 1]);
      const auto lo = __builtin_amdgcn_cvt_pkrtz(p[2 * i] - static_cast<float>(hi[0]), p[2 * i + 1] - static_cast<float>(hi[1]));
      r[i] = __builtin_bit_cast(unsigned, hi);
      r[2 + i] = __builtin_bit_cast(unsigned, lo);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned hi = cvt_pk_bf16(p[2 * i], p[2 * i + 1]);
      r[i] = hi;
      r[2 + i] = cvt_pk_bf16(p[2 * i] - lo_bf16(hi), p[2 * i + 1] - hi_bf16(hi));
    }
  }
  return r;
}

// Two weights rounded to 16 bits each, and their sum added to l.
template <bool F16>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(unsigned, ta_f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
  return cvt_pk_bf16(a, b);
}
template <bool F16>
__device__ __forceinline__ float add2(unsigned p, float l) {
  if constexpr (F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(ta_f16x2, p), ta_f16x2{1, 1}, l, false);
  return dot2_bf16(p, 0x3f803f80u, l);
}

// x[l], y[l] = a[l % 32], a[l % 32 + 32] (swap32), or a of the even and odd
// 16-lane row of l's pair (swap16): op(x, y) joins the lanes that hold one
// row's other keys. The s_nop covers the VALU-write to permlane-read hazard.
__device__ __forceinline__ void swap32(float a, float& x, float& y) {
  unsigned u = __builtin_bit_cast(unsigned, a), v = u;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(u), "+v"(v));
  x = __builtin_bit_cast(float, u);
  y = __builtin_bit_cast(float, v);
}
__device__ __forceinline__ void swap16(float a, float& x, float& y) {
  unsigned u = __builtin_bit_cast(unsigned, a), v = u;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(u), "+v"(v));
  x = __builtin_bit_cast(float, u);
  y = __builtin_bit_cast(float, v);
}
__device__ __forceinline__ float row_max(float a) {
  float x, y;
  swap32(a, x, y);
  a = fmaxf(x, y);
  swap16(a, x, y);
  return fmaxf(x, y);
}
__device__ __forceinline__ float row_sum(float a) {
  float x, y;
  swap32(a, x, y);
  a = x + y;
  swap16(a, x, y);
  return x + y;
}

// A weight is 2^(s c - m) with one rounding, while m is the largest s c rounded:
// the largest weight is 2^d instead of 1, d up to half a step of m. Sums and
// products carry the same factor, so that it cancels, as long as weights fit their
// 16 bits: fp16 takes them up to 2^14 lifted, so d may be 1 (m up to 2^24). A row
// whose maximum lies farther out (or is infinite) is done over by the join, which
// rounds every s c before it subtracts.
__device__ __forceinline__ bool far_out(float m) { return fabsf(m) > 0x1p24f && m != -INFINITY; }

// A word of memory that does not change during the launch, at a uniform
// address: a scalar load, which does not wait for the loads in flight.
__device__ __forceinline__ int uniform_word(const int* p, long long i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p))[i];
}

// The same value in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Inclusive prefix sum over the wave's lanes by DPP row shifts and broadcasts.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// Where the work is cut. A tile is R rows (node, head of the KV head's group)
// of one sequence and KV head; its units are kOver of them for starting and
// ending it, then one for each block of B keys: the cache's, then the tree's.
// Units are numbered sequence by sequence, and workgroup b takes units
// [b * chunk, (b + 1) * chunk): every workgroup gets the same share, however
// ragged the lengths; no fewer than 2 units (6 of the kernel of many rows), as
// more parts cost the join more than they save (one token behind 2047, smallest
// share 1, 2, 4, 8: 9.2, 8.6, 9.5, 11.3 us; 240 rows behind 2000 with 1, 4, 6, 8:
// 22.6, 18.0, 16.7, 18.4). The host sees to it that all units count in 31 bits.
constexpr int kOver = 3;

struct Tiles {
  int first, nodes, len, cached, blocks, row_tiles, units;
  __device__ __forceinline__ int tile_units() const { return blocks + kOver; }
};

template <int R, int B>
__device__ __forceinline__ Tiles tiles_from(const TreeArgs& a, int start, int stop, int len) {
  Tiles t;
  t.first = min(max(start, 0), a.num_nodes);
  t.nodes = min(min(max(stop, t.first), a.num_nodes) - t.first, a.max_nodes);
  t.len = min(max(len, 0), a.max_pages << a.page_shift);
  t.cached = (t.len + B - 1) / B;
  t.blocks = t.cached + (t.nodes + B - 1) / B;
  t.row_tiles = (t.nodes * a.G + R - 1) / R;
  t.units = t.row_tiles * a.Hkv * t.tile_units();
  return t;
}
template <int R, int B>
__device__ __forceinline__ Tiles tiles_of(const TreeArgs& a, int s) {
  return tiles_from<R, B>(a, a.starts[s], a.starts[s + 1], a.lens[s]);
}
// The same of a sequence that is one for the whole wave, by scalar loads.
template <int R, int B>
__device__ __forceinline__ Tiles uniform_tiles_of(const TreeArgs& a, int s) {
  return tiles_from<R, B>(a, uniform_word(a.starts, s), uniform_word(a.starts, s + 1), uniform_word(a.lens, s));
}

// The share of workgroup b: its units, the sequence of the first one and the
// units before that sequence. Every wave finds it by itself, without a barrier.
struct Share {
  int at, end, s, base;
  Tiles t;
};

template <int R, int B>
__device__ __forceinline__ bool share_of(const TreeArgs& a, int b, Share& sh) {
  const int lane = threadIdx.x & 63, per = (a.num_seqs + 63) / 64, s0 = lane * per;
  Tiles t = {};
  int mine = 0;
  for (int i = 0; i < per; ++i)
    if (s0 + i < a.num_seqs) {
      t = tiles_of<R, B>(a, s0 + i);
      mine += t.units;
    }
  const int incl = wave_scan(mine), total = __builtin_amdgcn_readlane(incl, 63);
  const int chunk = max(static_cast<int>((static_cast<unsigned>(total) + a.workgroups - 1) / a.workgroups), R == 128 ? 6 : 2);
  int at = incl - mine;
  if (b == 0 && threadIdx.x < 64) {  // for the launch that joins the parts
    int before = at;
    for (int i = 0; i < per; ++i)
      if (s0 + i < a.num_seqs) {
        a.prefix[s0 + i] = before;
        if (per > 1) before += tiles_of<R, B>(a, s0 + i).units;
      }
    if (lane == 0) a.prefix[a.num_seqs] = chunk;
  }
  const long long first = static_cast<long long>(b) * chunk;
  if (first >= total) return false;
  const int u = static_cast<int>(first);
  const bool has = at <= u && u < incl;
  int s = s0;
  if (has && per > 1)
    for (;; ++s) {
      t = tiles_of<R, B>(a, s);
      if (u < at + t.units) break;
      at += t.units;
    }
  const int who = __ffsll(static_cast<unsigned long long>(__ballot(has))) - 1;
  auto pick = [&](int x) { return __builtin_amdgcn_readlane(x, who); };
  sh.at = u;
  sh.end = static_cast<int>(min(first + chunk, static_cast<long long>(total)));
  sh.s = pick(s);
  sh.base = pick(at);
  sh.t = {pick(t.first), pick(t.nodes), pick(t.len), pick(t.cached), pick(t.blocks), pick(t.row_tiles), pick(t.units)};
  return true;
}

template <int D>
__device__ __forceinline__ int k_slot(int row, int c) {  // 16 rows of a 16-byte read on different banks
  return D == 64 ? c ^ ((row >> 1) & 7) : c ^ row;
}
template <int D>
__device__ __forceinline__ int v_slot(int row, int c) {  // the 8 rows of half a transposed read on different banks
  return D == 64 ? c ^ (((row >> 1) & 3) << 1) : c ^ ((row & 7) << 1);
}

template <int D>
__device__ __forceinline__ int wide_v_slot(int row, int c) {  // the 4 rows of half a wider transposed read
  return D == 64 ? c ^ (((row >> 1) & 1) << 2) : c ^ ((row & 3) << 2);
}

// A wave waits until at most N of its loads are in flight and its LDS reads
// are done: a stage has landed, and the one before it may be overwritten.
template <int N>
__device__ __forceinline__ void wait_stage() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

typedef float ta_f32x16 __attribute__((ext_vector_type(16)));

template <bool F16>
__device__ __forceinline__ ta_f32x16 mfma32(ta_u32x4 a, ta_u32x4 b, ta_f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ta_f16x8, a), __builtin_bit_cast(ta_f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ta_bf16x8, a), __builtin_bit_cast(ta_bf16x8, b), c, 0, 0, 0);
}

// Row (n, h) of sequence s by one wave, one key at a time and only the keys that
// have a weight (a product with a weight of zero lets what is not seen through).
template <int D, bool F16, bool I4>
__device__ __forceinline__ void attend_row(const TreeArgs& a, const Tiles& t, int s, int n, int h) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, hk = h / a.G;
  uint16_t* out = a.out + (static_cast<long long>(n) * a.H + h) * D;
  const uint16_t* q = a.q + (static_cast<long long>(n) * a.H + h) * D;
  const int ps = 1 << a.page_shift;
  // the key and value of position or node j, null where the row does not see it
  auto key = [&](int j, const uint16_t*& v) -> const uint16_t* {
    if (j < t.len) {
      const int page = a.table[static_cast<long long>(s) * a.max_pages + (j >> a.page_shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_pages)) return nullptr;
      const long long at = ((static_cast<long long>(page) * a.Hkv + hk) * ps + (j & (ps - 1))) * (I4 ? kInt4Row<D> / 2 : D);
      v = a.v_pages + at;
      return a.k_pages + at;
    }
    j -= t.len;
    if (j >= t.nodes || !(a.mask[static_cast<long long>(n) * a.words + (j >> 5)] >> (j & 31) & 1)) return nullptr;
    const long long at = (static_cast<long long>(t.first + j) * a.Hkv + hk) * D;
    v = a.v_new + at;
    return a.k_new + at;
  };
  const int keys = t.len + t.nodes;
  auto element = [&](const uint16_t* row, int j, int d) { return I4 && j < t.len ? int4_value<D>(row, d) : widen<F16>(row[d]); };
  auto score = [&](int j, const uint16_t*& v) {  // one key a lane; v null where it has no weight
    v = nullptr;
    const uint16_t* k = j < keys ? key(j, v) : nullptr;
    if (!k) return -INFINITY;
    float x = 0.f;
    for (int d = 0; d < D; ++d) x += widen<F16>(q[d]) * element(k, j, d);
    x *= a.scale_log2;
    if (x == -INFINITY) v = nullptr;
    return x;
  };
  float top = -INFINITY, sum = 0.f, o[E] = {};
  for (int j = 0; j < keys; j += 64) {
    const uint16_t* v;
    top = fmaxf(top, score(j + lane, v));
  }
  top = wave_max(top);
  auto weight = [&](float x, const uint16_t* v) {
    return !v ? 0.f : x != x || top == INFINITY ? NAN : __builtin_amdgcn_exp2f(x - top);
  };
  for (int j = 0; j < keys; j += 64) {
    const uint16_t* v;
    const float x = score(j + lane, v);
    sum += weight(x, v);
  }
  sum = wave_sum(sum);
  const float inv = 1.f / sum;
  if (sum == sum && sum != 0.f)
    for (int j = 0; j < keys; j += 64) {
      const uint16_t* v;
      const float x = score(j + lane, v), p = weight(x, v) * inv;  // divided first: sums of the largest values stay finite
      const unsigned long long seen = __ballot(v != nullptr);
      for (unsigned long long left = seen; left; left &= left - 1) {
        const int i = __ffsll(static_cast<unsigned long long>(left)) - 1;
        const float pi = __shfl(p, i, 64);
        const uintptr_t vi = static_cast<uintptr_t>(__shfl(static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(v)), i, 64));
        for (int e = 0; e < E; ++e) {
          const float x = element(reinterpret_cast<const uint16_t*>(vi), j + i, lane * E + e);
          // a weight too small for fp32 is still not zero: an infinity stays one
          o[e] += (__builtin_isinf(x) ? fmaxf(pi, 1.17549435e-38f) : pi) * x;
        }
      }
    }
  for (int e = 0; e < E; ++e) out[lane * E + e] = narrow<F16>(sum != sum ? NAN : o[e]);
}

// One workgroup per node and 4 heads, a wave for each row: joins the parts of
// rows whose keys were shared out, and does over the rows that came out
// infinite or NaN (or whose scores lie too far out: far_out).
template <int D, bool F16, int R, int B, bool I4>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
  constexpr int E = D / 64, V4 = D / 4, NP = 64 / V4;  // parts added at a time
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int n = blockIdx.x, h = blockIdx.y * 4 + w;
  const int s = uniform_word(a.owner, n);  // anything where no workgroup wrote it: checked like any number
  if (static_cast<unsigned>(s) >= static_cast<unsigned>(a.num_seqs) || h >= a.H) return;
  const Tiles t = uniform_tiles_of<R, B>(a, s);
  const int chunk = uniform_word(a.prefix, a.num_seqs), before = uniform_word(a.prefix, s);
  if (n < t.first || n >= t.first + t.nodes) return;
  const int G = a.G, hk = h / G, row = (n - t.first) * G + (h - hk * G);
  const int u0 = before + (hk * t.row_tiles + row / R) * t.tile_units() + kOver, u1 = u0 + t.blocks - 1;
  const int b0 = u0 / chunk, b1 = u1 / chunk;
  uint16_t* out = a.out + (static_cast<long long>(n) * a.H + h) * D;
  bool again = false;
  if (b0 == b1) {  // one workgroup had all its keys
    for (int e = 0; e < E; ++e) again |= !__builtin_isfinite(widen<F16>(out[lane * E + e]));
  } else {
    const int parts = b1 - b0 + 1;
    const long long r = row % R;
    auto slot = [&](int i) { return (2LL * (b0 + i) + (i == 0)) * R + r; };
    float2 ml = lane < parts ? a.part_ml[slot(lane)] : make_float2(-INFINITY, 0.f);
    const int g = lane / V4;
    constexpr int kAhead = 8;  // loads in flight
    ta_f32x4 x[kAhead];
    auto load = [&](int i) {  // parts i + g, i + g + NP, ..
#pragma unroll
      for (int k = 0; k < kAhead; ++k) x[k] = *reinterpret_cast<const ta_f32x4*>(a.part_o + slot(min(i + k * NP + g, parts - 1)) * D + (lane % V4) * 4);
    };
    load(0);  // with the maxima: one round trip for most rows
    float top = ml.x;
    for (int i = 64 + lane; i < parts; i += 64) top = fmaxf(top, a.part_ml[slot(i)].x);
    top = wave_max(top);
    again |= far_out(top);
    float sum = 0.f;
    ta_f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < parts; i0 += 64) {
      if (i0) ml = i0 + lane < parts ? a.part_ml[slot(i0 + lane)] : make_float2(-INFINITY, 0.f);
      // the weight of part i0 + lane, below 0 for a part that saw nothing. One too small
      // for fp32 is 0, and makes NaN of an infinite sum, which has the row done over.
      const float f = ml.y == 0.f ? -1.f : __builtin_amdgcn_exp2f(ml.x - top);
      sum += ml.y == 0.f ? 0.f : f * ml.y;
      for (int i = 0; i < min(parts - i0, 64); i += kAhead * NP) {
        if (i0 + i) load(i0 + i);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int j = i + k * NP + g;
          const float fj = __shfl(f, j, 64);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += fj < 0.f ? 0.f : fj * x[k][e];
        }
      }
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int d = V4; d < 64; d *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], d, 64);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (sum == 0.f) v = ta_f32x4{0.f, 0.f, 0.f, 0.f};
    ta_u32x2 y;
    for (int e = 0; e < 4; ++e) again |= !__builtin_isfinite(v[e] * inv);
    y.x = narrow<F16>(v[0] * inv) | static_cast<unsigned>(narrow<F16>(v[1] * inv)) << 16;
    y.y = narrow<F16>(v[2] * inv) | static_cast<unsigned>(narrow<F16>(v[3] * inv)) << 16;
    if (lane < V4) *reinterpret_cast<ta_u32x2*>(out + lane * 4) = y;
  }
  if (__builtin_amdgcn_ballot_w64(again)) attend_row<D, F16, I4>(a, t, s, n, h);
}

// Row tiles of 16, 32 or 128 rows. The kernel that splits a block's keys over
// its waves also ran tiles of 64, which lost to the kernel of many rows from 33
// rows on (40 rows behind 37-3968 positions, 8 sequences: 18.1 against 16.4 us;
// 64 rows behind 1000-3968, 16 sequences: 32.2 against 28.7; head_dim 128, 40 rows,
// 4 sequences: 24.5 against 21.1); at 17 to 32 rows the two are equal (23.6 against
// 24.3, head_dim 128 42.2 against 42.0) and this one keeps the weights' 16 bits.
int rows_of_tile(int n_heads, int n_kv_heads, int max_nodes) {
  const int rows = max_nodes * (n_heads / n_kv_heads);
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 128;
}

// Units of work that there can be at most.
long long most_units(int n_heads, int n_kv_heads, int num_seqs, int max_nodes, int max_pages, int page_size) {
  const int R = rows_of_tile(n_heads, n_kv_heads, max_nodes);
  const int B = R == 128 ? kWideBlock : kBlock;
  const long long blocks = (static_cast<long long>(max_pages) * page_size + B - 1) / B + (max_nodes + B - 1) / B;
  const long long tiles = static_cast<long long>((max_nodes * (n_heads / n_kv_heads) + R - 1) / R) * n_kv_heads * num_seqs;
  return tiles * (blocks + kOver);
}

constexpr int kMaxNodes = 1024;

const char* check_shape(int n_heads, int n_kv_heads, int head_dim, int num_seqs, int num_nodes, int max_nodes,
                        int max_pages, int page_size) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads) return "n_heads must be a multiple of n_kv_heads";
  if (n_heads > 1024) return "n_heads exceeds 1024";
  if (num_seqs < 1 || num_seqs > 8192) return "num_seqs outside [1, 8192]";
  if (num_nodes < 1 || num_nodes > (1 << 20)) return "num_nodes outside [1, 2^20]";
  if (max_nodes < 1 || max_nodes > kMaxNodes) return "max_nodes outside [1, 1024]";
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return "page_size is not a power of two from 16 to 1024";
  if (max_pages < 1 || static_cast<long long>(max_pages) * page_size >= (1LL << 31) - (1 << 20))
    return "max_pages: a sequence holds less than 2^31 - 2^20 positions";
  if (most_units(n_heads, n_kv_heads, num_seqs, max_nodes, max_pages, page_size) >= (1LL << 31))
    return "num_seqs * max_pages * page_size * row tiles is too large: blocks of 32 keys must count below 2^31";
  return nullptr;
}

// The workspace of a call whose kernels run on `resident(D, R)` workgroups at once.
typedef int (*Resident)(int D, int R);

int workgroups_of(Resident resident, int n_heads, int n_kv_heads, int head_dim, int num_seqs, int max_nodes, int max_pages,
                  int page_size) {
  return static_cast<int>(std::min<long long>(most_units(n_heads, n_kv_heads, num_seqs, max_nodes, max_pages, page_size), resident(head_dim, rows_of_tile(n_heads, n_kv_heads, max_nodes))));
}

long long tree_workspace(Resident resident, int n_heads, int n_kv_heads, int head_dim, int num_seqs, int num_nodes,
                         int max_nodes, int max_pages, int page_size) {
  if (check_shape(n_heads, n_kv_heads, head_dim, num_seqs, num_nodes, max_nodes, max_pages, page_size)) return -1;
  const long long slots = 2LL * workgroups_of(resident, n_heads, n_kv_heads, head_dim, num_seqs, max_nodes, max_pages, page_size) *
                          rows_of_tile(n_heads, n_kv_heads, max_nodes);
  return slots * head_dim * 4 + slots * 8 + (num_seqs + 1 + num_nodes) * 4LL;
}

// Checks a call and fills its arguments.
int tree_call(const char* who, Resident resident, TreeArgs& a, const void* q, const void* k_new, const void* v_new, const void* k_pages,
              const void* v_pages, const int* page_table, const int* seq_lens, const int* node_starts,
              const int* tree_mask, void* out, int dtype, int n_heads, int n_kv_heads, int head_dim, int num_pages,
              int page_size, int num_seqs, int max_pages, int num_nodes, int max_nodes, float scale, void* workspace,
              long long workspace_bytes) {
  const char* bad = check_shape(n_heads, n_kv_heads, head_dim, num_seqs, num_nodes, max_nodes, max_pages, page_size);
  IRON_REQUIRE(!bad, "%s: %s", who, bad);
  IRON_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype=%d is neither 0 (bf16) nor 1 (fp16)", who, dtype);
  IRON_REQUIRE(num_pages >= 1 && num_pages <= (1 << 27), "%s: num_pages=%d outside [1, 2^27]", who, num_pages);
  for (const void* p : {q, k_new, v_new, k_pages, v_pages, static_cast<const void*>(out)})
    IRON_REQUIRE(p && aligned16(p), "%s: null pointer, or one that is not 16-byte aligned", who);
  for (const void* p : {page_table, seq_lens, node_starts, tree_mask})
    IRON_REQUIRE(p && (reinterpret_cast<uintptr_t>(p) & 3u) == 0, "%s: int32 arrays must be given and 4-byte aligned", who);
  for (const void* p : {q, k_new, v_new, k_pages, v_pages}) IRON_REQUIRE(out != p, "%s: out is one of the inputs", who);
  IRON_REQUIRE(scale > 0.f && scale <= 1e30f, "%s: scale=%g must be positive and at most 1e30", who, scale);
  const long long need = tree_workspace(resident, n_heads, n_kv_heads, head_dim, num_seqs, num_nodes, max_nodes, max_pages, page_size);
  IRON_REQUIRE(workspace && aligned16(workspace), "%s: the workspace must be given and 16-byte aligned", who);
  IRON_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes, %lld needed", who, workspace_bytes, need);
  a.q = static_cast<const uint16_t*>(q);
  a.k_new = static_cast<const uint16_t*>(k_new);
  a.v_new = static_cast<const uint16_t*>(v_new);
  a.k_pages = static_cast<const uint16_t*>(k_pages);
  a.v_pages = static_cast<const uint16_t*>(v_pages);
  a.table = page_table;
  a.lens = seq_lens;
  a.starts = node_starts;
  a.mask = tree_mask;
  a.out = static_cast<uint16_t*>(out);
  a.H = n_heads;
  a.Hkv = n_kv_heads;
  a.G = n_heads / n_kv_heads;
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctz(page_size);
  a.num_seqs = num_seqs;
  a.max_pages = max_pages;
  a.num_nodes = num_nodes;
  a.max_nodes = max_nodes;
  a.words = (max_nodes + 31) / 32;
  a.scale_log2 = scale * 1.4426950408889634f;
  const int R = rows_of_tile(n_heads, n_kv_heads, max_nodes);
  a.workgroups = workgroups_of(resident, n_heads, n_kv_heads, head_dim, num_seqs, max_nodes, max_pages, page_size);
  const long long slots = 2LL * a.workgroups * R;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * head_dim);
  a.prefix = reinterpret_cast<int*>(a.part_ml + slots);
  a.owner = a.prefix + num_seqs + 1;
  return 0;
}

}  // namespace
}  // namespace iron
