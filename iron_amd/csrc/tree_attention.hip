// Attention of drafted trees over a paged KV cache.
//
// out[i,h] = sum_j softmax_j(scale q[i,h] . k_j) v_j over the cached positions
// of node i's sequence and the nodes of its tree that it sees. The rows that
// share a KV head (nodes times heads of its group) make the tiles of a sequence,
// so that a byte of the cache is read once for all of them.
//
// Three launches' worth of code, two of them in a call:
//  - tree_attention_kernel, tiles of 16 or 32 rows: a decode step, a small tree.
//    Bound by the cache's bytes. Every wave streams its own keys through its own
//    LDS ring, without barriers.
//  - tree_wide_kernel, tiles of 128 rows: bound by the softmax and the products
//    together. The four waves share a ring.
//  - tree_join_kernel joins what different workgroups made of one row's keys.
// The work is cut into equal shares of key blocks whatever the lengths
// (share_of), from device memory alone: one captured graph serves every step.
//
// Measured (32 / 8 heads, whole calls back to back; a large copy moves 4.74 TB/s,
// a large library product does 1.14-1.17 PFLOP/s): 64 sequences of 150-16384
// positions, one token each, head_dim 64: 94 us, 5.1 TB/s of cache; the same with
// a cache that fits L2: 47 us. One token behind 2047: 12.6 us, 8.6 in a graph.
// 8 trees of 26 nodes behind 37-3968: 18.6 us. 2 trees of 64 nodes behind 20011 and
// 32768, head_dim 128, fp16: 99-109 us, 530-580 TFLOP/s; 93 with a cache that fits L2.
#include "iron_common.hpp"
#include "../../include/iron_hip.h"

#include <algorithm>
#include <type_traits>

namespace iron {
namespace {

struct TreeArgs {
  const uint16_t* q;        // (num_nodes, H, D)
  const uint16_t* k_new;    // (num_nodes, Hkv, D)
  const uint16_t* v_new;
  const uint16_t* k_pages;  // (num_pages, Hkv, page_size, D)
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

// The tree of sequence s: its first row and its nodes, cut to the arrays.
__device__ __forceinline__ void tree_of(const TreeArgs& a, int s, int& first, int& nodes) {
  first = min(max(a.starts[s], 0), a.num_nodes);
  nodes = min(min(max(a.starts[s + 1], first), a.num_nodes) - first, a.max_nodes);
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

// Few rows: a tile of 16 RT rows, a workgroup of 4 waves. Wave w has keys 16 w ..
// + 15 of each block of 64 and all rows, so nothing is shared until the end: each
// wave fills a ring of its own (LDS-direct loads, three blocks in flight, 96 KiB a
// CU) and waits for its own loads only. S^T = K Q^T on 16x16x32 MFMAs leaves each
// lane 4 keys of one row; as hi and lo halves (split4) they are the 8 elements of
// the B operand of O^T += V^T P^T as they stand, with V^T's 4 keys given twice, from
// one transposed LDS read. The waves' sums meet in LDS once per tile.
template <int D, bool F16, int RT>
__global__ __launch_bounds__(256) void tree_attention_kernel(TreeArgs a) {
  constexpr int R = 16 * RT, B = kBlock, kRow = D * 2, kHalf = 16 * kRow, kStage = 2 * kHalf, kRing = kStages * kStage;
  constexpr int kLoads = kStage / 1024;  // 1 KiB loads of a stage, the first half of them K
  constexpr int NK = D / 32, ND = D / 16;
  static_assert(R * D * 4 <= kRing, "a wave's output goes through its ring");
  __shared__ __attribute__((aligned(16))) unsigned char lds[4 * kRing];
  __shared__ float stat_m[4][R], stat_l[4][R];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int c = lane & 15, quad = lane >> 4;
  const int G = a.G, ps = 1 << a.page_shift;
  Share sh;
  if (!share_of<R, B>(a, blockIdx.x, sh)) return;
  int u = sh.at, s = sh.s, base = sh.base;
  const int end = sh.end;
  Tiles t = sh.t;

  // This lane's part of a stage's loads: load i puts 1024 bytes, 16 from each
  // lane in order, so lane l fetches the chunk that belongs at its slot.
  int lrow[kLoads / 2];
  unsigned kchunk[kLoads / 2], vchunk[kLoads / 2];
#pragma unroll
  for (int i = 0; i < kLoads / 2; ++i) {
    const int slot = lane % (kRow / 16), row = i * (1024 / kRow) + lane / (kRow / 16);
    lrow[i] = row;
    kchunk[i] = k_slot<D>(row, slot) * 16;
    vchunk[i] = v_slot<D>(row, slot) * 16;
  }
  unsigned char* ring = lds + w * kRing;
  const int trow = 4 * quad + (c >> 2), tcol = 4 * (c & 3);  // this lane's address of a transposed V read

  while (u < end) {
    const int tu = t.tile_units(), tile = uniform((u - base) / tu), in_tile = (u - base) - tile * tu;
    const int stop = min(tu, in_tile + (end - u)), blk0 = max(in_tile - kOver, 0), n = stop - kOver - blk0;
    const int hk = uniform(tile / t.row_tiles), row0 = (tile - hk * t.row_tiles) * R;
    const int rows = min(R, t.nodes * G - row0);
    if (n > 0) {
      if (hk == 0 && blk0 == 0)  // for the launch that joins the parts
        for (int i = row0 / G + tid; i <= (row0 + rows - 1) / G; i += 256) a.owner[t.first + i] = s;
      ta_u32x4 qf[RT][NK];
      int node[RT];
      ta_f32x4 o[RT][ND];
      float m[RT], off[RT], l[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        off[rt] = l[rt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[rt][dt] = ta_f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const long long table = static_cast<long long>(s) * a.max_pages;
      const unsigned new_row = static_cast<unsigned>(a.Hkv) * kRow;
      unsigned holes = 0;  // bit i % kStages: block i's page of this wave is none
      auto page_of = [&](int i) {
        const int blk = min(blk0 + i, t.cached - 1);
        return t.cached ? uniform_word(a.table, table + (min(blk * kBlock + 16 * w, t.len - 1) >> a.page_shift)) : 0;
      };
      // the pages of the blocks that are issued next, read ahead: one round trip for the first ones
      int page[kStages];
#pragma unroll
      for (int i = 0; i < kStages; ++i) page[i] = page_of(i);
      auto issue = [&](int i) {
        unsigned char* st = ring + (i % kStages) * kStage;
        const int blk = blk0 + i;
        if (blk < t.cached) {
          const bool real = static_cast<unsigned>(page[0]) < static_cast<unsigned>(a.num_pages);
          holes = (holes & ~(1u << (i % kStages))) | (real ? 0u : 1u << (i % kStages));
          const long long at = ((static_cast<long long>(real ? page[0] : 0) * a.Hkv + hk) * ps + ((blk * kBlock + 16 * w) & (ps - 1))) * D;
          const i32x4v rk = buffer_rsrc(a.k_pages + at), rv = buffer_rsrc(a.v_pages + at);
#pragma unroll
          for (int j = 0; j < kLoads / 2; ++j) {
            load_lds16(rk, lrow[j] * kRow + kchunk[j], st + j * 1024);
            load_lds16(rv, lrow[j] * kRow + vchunk[j], st + kHalf + j * 1024);
          }
#pragma unroll
          for (int j = 0; j + 1 < kStages; ++j) page[j] = page[j + 1];
          page[kStages - 1] = page_of(i + kStages);
        } else {
          const int j0 = (blk - t.cached) * kBlock + 16 * w;
          const long long at = (static_cast<long long>(t.first) * a.Hkv + hk) * D;
          const i32x4v rk = buffer_rsrc(a.k_new + at), rv = buffer_rsrc(a.v_new + at);
#pragma unroll
          for (int j = 0; j < kLoads / 2; ++j) {
            const unsigned r = min(j0 + lrow[j], t.nodes - 1) * new_row;
            load_lds16(rk, r + kchunk[j], st + j * 1024);
            load_lds16(rv, r + vchunk[j], st + kHalf + j * 1024);
          }
        }
      };

      auto step = [&](int i) {
        const int blk = blk0 + i;
        const bool cache = blk < t.cached;
        const int j0 = (cache ? blk : blk - t.cached) * kBlock + 16 * w;
        const int valid = cache && (holes >> (i % kStages) & 1) ? 0 : min((cache ? t.len : t.nodes) - j0, 16);
        if (valid <= 0) return;
        const unsigned char* ks = ring + (i % kStages) * kStage;
        const unsigned char* vs = ks + kHalf;
        ta_u32x4 kf[NK];
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) kf[kk] = *reinterpret_cast<const ta_u32x4*>(ks + c * kRow + k_slot<D>(c, 4 * kk + quad) * 16);
        ta_u32x2 vt[ND];
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const int dim = 16 * dt + tcol;
          vt[dt] = __builtin_bit_cast(ta_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) ta_i16x4*)(vs + trow * kRow + v_slot<D>(trow, dim >> 3) * 16 + (dim & 7) * 2)));
        }
        ta_f32x4 sc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          sc[rt] = ta_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) sc[rt] = mfma<F16>(kf[kk], qf[rt][kk], sc[rt]);
        }
        if (valid < 16) {  // keys behind the last one: no score, and values that cannot do harm
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][e] = 4 * quad + e < valid ? sc[rt][e] : -INFINITY;
          const unsigned k0 = 4 * quad;
          const unsigned m01 = (k0 < static_cast<unsigned>(valid) ? 0xffffu : 0u) | (k0 + 1 < static_cast<unsigned>(valid) ? 0xffff0000u : 0u);
          const unsigned m23 = (k0 + 2 < static_cast<unsigned>(valid) ? 0xffffu : 0u) | (k0 + 3 < static_cast<unsigned>(valid) ? 0xffff0000u : 0u);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) {
            vt[dt].x &= m01;
            vt[dt].y &= m23;
          }
        }
        if (!cache) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const int word = a.mask[static_cast<long long>(node[rt]) * a.words + (j0 >> 5)] >> ((j0 & 31) + 4 * quad);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[rt][e] = word >> e & 1 ? sc[rt][e] : -INFINITY;
          }
        }
        // Softmax in the log2 domain, p = 2^(s c - m). The row's maximum m moves only
        // when a score passes it by more than 8, so p <= 2^8 and O is rarely
        // rescaled; sum(p v) / sum(p) does not depend on which m is used.
        const float cs = a.scale_log2;
        bool grow = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          grow |= fmaxf(fmaxf(sc[rt][0], sc[rt][1]), fmaxf(sc[rt][2], sc[rt][3])) * cs > m[rt] + 8.f;
        if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const float top = row_max(fmaxf(fmaxf(sc[rt][0], sc[rt][1]), fmaxf(sc[rt][2], sc[rt][3]))) * cs;
            if (top > m[rt] + 8.f) {
              const float alpha = __builtin_amdgcn_exp2f(m[rt] - top);  // 0 from m = -inf
              m[rt] = top;
              off[rt] = top - kLift<F16>;
              l[rt] *= alpha;
#pragma unroll
              for (int dt = 0; dt < ND; ++dt) o[rt][dt] *= alpha;
            }
          }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[rt][e], cs, -off[rt]));
          l[rt] += (p[0] + p[1]) + (p[2] + p[3]);
          const ta_u32x4 pf = split4<F16>(p);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) o[rt][dt] = mfma<F16>(ta_u32x4{vt[dt].x, vt[dt].y, vt[dt].x, vt[dt].y}, pf, o[rt][dt]);
        }
      };

      static_assert(kStages == 4, "the waits below count three stages in flight");
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i)
        if (i < n) issue(i);
      // Q: the B operand of S^T = K Q^T (column: row 16 rt + c; dims 32 kk + 8 quad .. + 8).
      // The compiler's wait for it takes in the ring's first loads, which it does not
      // count: one round trip for both.
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = min(row0 + 16 * rt + c, t.nodes * G - 1), in_tree = r / G;
        node[rt] = t.first + in_tree;
        const uint16_t* qp = a.q + (static_cast<long long>(node[rt]) * a.H + hk * G + (r - in_tree * G)) * D + 8 * quad;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[rt][kk] = *reinterpret_cast<const ta_u32x4*>(qp + 32 * kk);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) asm volatile("" ::"v"(qf[rt][kk]));
      for (int i = 0; i < n; ++i) {
        const int left = n - 1 - i;  // stages in flight behind block i
        if (left >= 2)
          wait_stage<2 * kLoads>();
        else if (left == 1)
          wait_stage<kLoads>();
        else
          wait_stage<0>();
        if (i + kStages - 1 < n) issue(i + kStages - 1);  // into the stage of block i - 1, which every read has left
        step(i);
      }

      // The four waves' parts of the tile meet in LDS.
      const bool whole = n == t.blocks;
      const long long slot = 2LL * blockIdx.x + (blk0 == 0 ? 1 : 0);
      wait_stage<0>();
      float* mine_o = reinterpret_cast<float*>(ring);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = 16 * rt + c;
        const float sum = row_sum(l[rt]);
        if (quad == 0) {
          stat_m[w][r] = m[rt] - kLift<F16>;
          stat_l[w][r] = sum;
        }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
          *reinterpret_cast<ta_f32x4*>(mine_o + r * D + (((4 * dt + quad) ^ c) * 4)) = o[rt][dt];
      }
      __syncthreads();
      for (int x = tid; x < rows * (D / 4); x += 256) {
        const int r = x / (D / 4), c4 = x % (D / 4);
        float top = stat_m[0][r];
#pragma unroll
        for (int i = 1; i < 4; ++i) top = fmaxf(top, stat_m[i][r]);
        float sum = 0.f;
        ta_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float li = stat_l[i][r];
          const float f = __builtin_amdgcn_exp2f(stat_m[i][r] - top);
          const ta_f32x4 part = f * *reinterpret_cast<const ta_f32x4*>(reinterpret_cast<const float*>(lds + i * kRing) + r * D + ((c4 ^ (r & 15)) * 4));
          sum += li == 0.f ? 0.f : f * li;  // a wave that saw nothing has no maximum either
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += li == 0.f ? 0.f : part[e];
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          ta_u32x2 y;
          if (sum == 0.f) v = ta_f32x4{0.f, 0.f, 0.f, 0.f};
          if (far_out(top)) v = ta_f32x4{NAN, NAN, NAN, NAN};  // for the launch that joins the parts
          y.x = narrow<F16>(v[0] * inv) | static_cast<unsigned>(narrow<F16>(v[1] * inv)) << 16;
          y.y = narrow<F16>(v[2] * inv) | static_cast<unsigned>(narrow<F16>(v[3] * inv)) << 16;
          const int row = row0 + r;
          *reinterpret_cast<ta_u32x2*>(a.out + (static_cast<long long>(t.first + row / G) * a.H + hk * G + row % G) * D + c4 * 4) = y;
        } else {
          *reinterpret_cast<ta_f32x4*>(a.part_o + (slot * R + r) * D + c4 * 4) = v;
          if (c4 == 0) a.part_ml[slot * R + r] = make_float2(top, sum);
        }
      }
      __syncthreads();  // the rings are free again
    }
    u += stop - in_tile;
    if (u < end && u == base + t.units) {
      base += t.units;
      do t = uniform_tiles_of<R, B>(a, ++s);
      while (t.units == 0);
    }
  }
}

typedef float ta_f32x16 __attribute__((ext_vector_type(16)));

template <bool F16>
__device__ __forceinline__ ta_f32x16 mfma32(ta_u32x4 a, ta_u32x4 b, ta_f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ta_f16x8, a), __builtin_bit_cast(ta_f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ta_bf16x8, a), __builtin_bit_cast(ta_bf16x8, b), c, 0, 0, 0);
}

// Many rows: a tile of 128 rows, a workgroup of 4 waves with 32 rows each. The
// waves load blocks of 32 keys together (8 rows of K and of V each) into one
// ring: every byte read from L2 serves 128 rows. One barrier per block; a SIMD's
// two waves (three with head_dim 64) are of different workgroups. Weights are
// rounded once, to the 16 bits of their type, as the prompt's attention (MHA)
// rounds them, and their sum is that of the rounded ones: as hi and lo they doubled the second
// product (134 -> 109 us for the wide trees above, with the next block's
// scores computed among this one's softmax; error against 64 bits 1.2 times that of
// one rounding of the result). What bounds it, by counters (the wide trees, fp16 and
// bf16 alike): of its SIMDs' cycles the matrix units are busy in 40 % and VALU
// instructions take 32 %, 72 % if they never meet; a wave waits for data or a
// barrier in 27 % of its time and to issue in another 27 %. Neither unit is full and
// two waves to a SIMD do not keep them both at work. Six of eight products of the
// second GEMM taken out saved 12 of 93 us, half of K's or V's LDS reads nothing,
// scheduling barriers, wave priorities and accumulators in AGPRs nothing.
template <int D, bool F16>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void tree_wide_kernel(TreeArgs a) {
  constexpr int R = 128, B = kWideBlock, kRow = D * 2, kHalf = B * kRow, kStage = 2 * kHalf;
  constexpr int kParts = 8 * kRow / 1024, kLoads = 2 * kParts;  // 1 KiB loads of a wave and block: kParts of K, kParts of V
  constexpr int NK = D / 16, ND = D / 32;
  __shared__ __attribute__((aligned(16))) unsigned char ring[kStages * kStage];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  const int G = a.G, ps = 1 << a.page_shift;
  Share sh;
  if (!share_of<R, B>(a, blockIdx.x, sh)) return;
  int u = sh.at, s = sh.s, base = sh.base;
  const int end = sh.end;
  Tiles t = sh.t;

  // This lane's 16 bytes of each of the wave's loads: rows 8 w .. + 7 of a block.
  unsigned krow[kParts], kat[kParts], vat[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int slot = lane % (kRow / 16), row = 8 * w + i * (1024 / kRow) + lane / (kRow / 16);
    krow[i] = row;
    kat[i] = k_slot<D>(row & 15, slot) * 16;
    vat[i] = wide_v_slot<D>(row, slot) * 16;
  }
  const int trow = 4 * hh + ((lane & 15) >> 2), tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const unsigned page_bytes = static_cast<unsigned>(a.Hkv) << a.page_shift << (D == 64 ? 7 : 8);

  while (u < end) {
    const int tu = t.tile_units(), tile = uniform((u - base) / tu), in_tile = (u - base) - tile * tu;
    const int stop = min(tu, in_tile + (end - u)), blk0 = max(in_tile - kOver, 0), n = stop - kOver - blk0;
    const int hk = uniform(tile / t.row_tiles), row0 = (tile - hk * t.row_tiles) * R;
    const int rows = min(R, t.nodes * G - row0);
    if (n > 0) {
      if (hk == 0 && blk0 == 0)  // for the launch that joins the parts
        for (int i = row0 / G + tid; i <= (row0 + rows - 1) / G; i += 256) a.owner[t.first + i] = s;
      const int* table = a.table + static_cast<long long>(s) * a.max_pages;
      const int cached = t.cached - blk0;                       // blocks of this part that are the cache's (the rest are the tree's)
      const int whole_blocks = t.len / B - blk0;                // the first ones of them, with no key behind the last
      const long long head = static_cast<long long>(hk) * ps * kRow;
      const unsigned char* kc = reinterpret_cast<const unsigned char*>(a.k_pages) + head;
      const unsigned char* vc = reinterpret_cast<const unsigned char*>(a.v_pages) + head;
      const long long tree = (static_cast<long long>(t.first) * a.Hkv + hk) * kRow;
      const unsigned new_row = static_cast<unsigned>(a.Hkv) * kRow;
      unsigned holes = 0;  // bits 2 (i % kStages) and + 1: the two pages of block i's 16 rows each are none
      // the pages of the blocks that are issued next, read ahead: one round trip for the first ones
      int page0[kStages] = {}, page1[kStages] = {};
      auto pages_of = [&](int i, int& p0, int& p1) {
        if (cached <= 0) return;
        const int pos = (blk0 + min(i, cached - 1)) * B;
        p0 = uniform_word(table, pos >> a.page_shift);
        p1 = uniform_word(table, min(pos + 16, t.len - 1) >> a.page_shift);
      };
#pragma unroll
      for (int i = 0; i < kStages; ++i) pages_of(i, page0[i], page1[i]);
      auto issue = [&](int i) {
        const int stage = i % kStages;
        unsigned char* st = ring + stage * kStage + 8 * w * kRow;
        if (i < cached) {
          const bool none0 = static_cast<unsigned>(page0[0]) >= static_cast<unsigned>(a.num_pages);
          const bool none1 = static_cast<unsigned>(page1[0]) >= static_cast<unsigned>(a.num_pages);
          holes = (holes & ~(3u << (2 * stage))) | ((none0 ? 1u : 0u) | (none1 ? 2u : 0u)) << (2 * stage);
          const unsigned page = w < 2 ? (none0 ? 0 : page0[0]) : (none1 ? 0 : page1[0]);
          // from the page's row of the block's first key: row 8 w is in the page, whatever page the first is in
          const int in_page = (((blk0 + i) * B + 8 * w) & (ps - 1)) - 8 * w;
          const long long at = static_cast<long long>(static_cast<unsigned long long>(page) * page_bytes) + in_page * kRow;
          const i32x4v rk = buffer_rsrc(kc + at), rv = buffer_rsrc(vc + at);
#pragma unroll
          for (int j = 0; j < kParts; ++j) {
            load_lds16(rk, krow[j] * kRow + kat[j], st + j * 1024);
            load_lds16(rv, krow[j] * kRow + vat[j], st + kHalf + j * 1024);
          }
#pragma unroll
          for (int j = 0; j + 1 < kStages; ++j) {
            page0[j] = page0[j + 1];
            page1[j] = page1[j + 1];
          }
          pages_of(i + kStages, page0[kStages - 1], page1[kStages - 1]);
        } else {
          const int j0 = (i - cached) * B;
          holes &= ~(3u << (2 * stage));
          const i32x4v rk = buffer_rsrc(reinterpret_cast<const unsigned char*>(a.k_new) + tree);
          const i32x4v rv = buffer_rsrc(reinterpret_cast<const unsigned char*>(a.v_new) + tree);
#pragma unroll
          for (int j = 0; j < kParts; ++j) {
            const unsigned r = min(j0 + static_cast<int>(krow[j]), t.nodes - 1) * new_row;
            load_lds16(rk, r + kat[j], st + j * 1024);
            load_lds16(rv, r + vat[j], st + kHalf + j * 1024);
          }
        }
      };
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i)
        if (i < n) issue(i);
      // Q: the B operand of S^T = K Q^T (column: row 32 w + c; dims 16 kk + 8 hh .. + 8)
      ta_u32x4 qf[NK];
      const int r = min(row0 + 32 * w + c, t.nodes * G - 1), in_tree = r / G;
      const int node = t.first + in_tree;
      const long long q_row = static_cast<long long>(node) * a.H + hk * G + (r - in_tree * G);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) qf[kk] = *reinterpret_cast<const ta_u32x4*>(a.q + q_row * D + 16 * kk + 8 * hh);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) asm volatile("" ::"v"(qf[kk]));
      ta_f32x16 o[ND];
      float m = -INFINITY, off = 0.f, l = 0.f;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[db][j] = 0.f;
      const bool idle = 32 * w >= rows;  // none of the wave's rows is one

      // Both swizzles are exclusive ors, so a fragment's address is the first one's with
      // the fragment's own bits turned: one register for each operand.
      const unsigned k_first = c * kRow + k_slot<D>(c & 15, hh) * 16;
      const unsigned v_first = kHalf + trow * kRow + wide_v_slot<D>(trow, tcol >> 3) * 16 + (tcol & 7) * 2;
      auto k_frag = [&](int i, int kk) {
        return *reinterpret_cast<const ta_u32x4*>(ring + (((i % kStages) * kStage + k_first) ^ (32 * kk)));
      };
      // V^T of keys 8 q + 4 hh .. + 3 of block i, dims 32 db + lane % 32
      auto v_frag = [&](int i, int q, int db) {
        return __builtin_bit_cast(ta_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ta_i16x4*)(
            ring + (((i % kStages) * kStage + v_first) ^ (64 * db)) + 8 * q * kRow)));
      };
      // The row's maximum, when scores pass it by more than 8 (in the log2 domain; cf. tree_attention_kernel).
      const float cs = a.scale_log2;
      auto raise = [&](const ta_f32x16& sc) {
        float mx = fmaxf(fmaxf(sc[0], sc[1]), sc[2]);
#pragma unroll
        for (int j = 3; j < 15; j += 2) mx = fmaxf(fmaxf(mx, sc[j]), sc[j + 1]);
        mx = fmaxf(mx, sc[15]);
        if (__builtin_amdgcn_ballot_w64(mx * cs > m + 8.f)) {
          float x, y;
          swap32(mx, x, y);
          const float top = fmaxf(x, y) * cs;
          if (top > m + 8.f) {
            const float alpha = __builtin_amdgcn_exp2f(m - top);  // 0 from m = -inf
            m = top;
            off = top - kLift<F16>;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < ND; ++db) o[db] *= alpha;
          }
        }
      };
      // Weights 2 g and 2 g + 1 of the lane, rounded to 16 bits as the second product takes them; l sums those.
      auto weights = [&](const ta_f32x16& sc, int g) {
        const unsigned p = pack2<F16>(__builtin_amdgcn_exp2f(fmaf(sc[2 * g], cs, -off)), __builtin_amdgcn_exp2f(fmaf(sc[2 * g + 1], cs, -off)));
        l = add2<F16>(p, l);
        return p;
      };
      // Block i from its scores S^T: sc[j] is key 8 (j / 4) + 4 hh + j % 4, row 32 w + c.
      auto step = [&](int i, ta_f32x16& sc, ta_f32x16& next) {
        const unsigned none = holes >> (2 * (i % kStages)) & 3u;
        if (i >= whole_blocks || none) {  // some of its keys are none, or not for every row
          const bool cache = i < cached;
          const int j0 = cache ? (blk0 + i) * B : (i - cached) * B, left = (cache ? t.len : t.nodes) - j0;
          unsigned keys = left >= 32 ? ~0u : (1u << left) - 1;  // those that there are
          keys &= ~((none & 1 ? 0xffffu : 0u) | (none & 2 ? 0xffff0000u : 0u));
          unsigned seen = keys;
          if (!cache) seen &= a.mask[static_cast<long long>(node) * a.words + (j0 >> 5)];
          seen >>= 4 * hh;
#pragma unroll
          for (int j = 0; j < 16; ++j) sc[j] = seen >> (8 * (j >> 2) + (j & 3)) & 1 ? sc[j] : -INFINITY;
          // The values of the others cannot do harm: every wave clears them before it
          // reads any (the waves write the same zeros, and none needs another's).
          for (int e = lane; e < B * (kRow / 16); e += 64)
            if (!(keys >> (e / (kRow / 16)) & 1))
              *reinterpret_cast<ta_u32x4*>(ring + (i % kStages) * kStage + kHalf + e * 16) = ta_u32x4{0, 0, 0, 0};
        }
        ta_u32x4 kf[NK];  // of block i + 1 (behind the last block: a stage that nothing writes, for scores that go unused)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) kf[kk] = k_frag(i + 1, kk);
        raise(sc);
        // In eight groups, held in this order by the scheduling barriers: two weights,
        // a part of V^T's reads, a product of the next block's scores, and from the
        // fifth on the products of the first 16 keys' weights. Left to itself the
        // compiler waits for each fragment of K before its product and puts the
        // exponentials behind all of them.
        ta_u32x4 pf[2];  // P^T of keys 16 g + 4 hh .. + 3 and + 8 .. + 11
        ta_u32x2 vt[4][ND];
        auto pv = [&](int g, int db) {
          o[db] = mfma32<F16>(ta_u32x4{vt[2 * g][db].x, vt[2 * g][db].y, vt[2 * g + 1][db].x, vt[2 * g + 1][db].y}, pf[g], o[db]);
        };
        next = ta_f32x16{};
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          __builtin_amdgcn_sched_barrier(0);
          if (g < NK) next = mfma32<F16>(kf[g], qf[g], next);
          if (g >= 4 && g - 4 < ND) pv(0, g - 4);
#pragma unroll
          for (int e = g * ND / 2; e < (g + 1) * ND / 2; ++e) vt[e / ND][e % ND] = v_frag(i, e / ND, e % ND);
          pf[g / 4][g % 4] = weights(sc, g);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int db = 0; db < ND; ++db) pv(1, db);
      };
      // Stages: i (V being read), i + 1 (K being read), i + 2 in flight, i + 3 being
      // issued into the one that every wave has left.
      auto turn = [&](int i, ta_f32x16& sc, ta_f32x16& next) {
        if (i + 1 < n) {
          if (i + 2 < n)
            wait_stage<kLoads>();
          else
            wait_stage<0>();
          __builtin_amdgcn_s_barrier();  // block i + 1 is there, and block i - 1's stage read by all
          asm volatile("" ::: "memory");
          if (i + kStages - 1 < n) issue(i + kStages - 1);
        }
        if (!idle) step(i, sc, next);
      };
      if (n >= 3)
        wait_stage<2 * kLoads>();
      else if (n == 2)
        wait_stage<kLoads>();
      else
        wait_stage<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      ta_f32x16 sa = {}, sb = {};
      if (!idle)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) sa = mfma32<F16>(k_frag(0, kk), qf[kk], sa);
      for (int i = 0; i < n; i += 2) {
        turn(i, sa, sb);
        if (i + 1 < n) turn(i + 1, sb, sa);
      }

      const bool whole = n == t.blocks;
      float l0, l1;
      swap32(l, l0, l1);
      const float sum = l0 + l1;
      const bool far = whole && far_out(m);  // NaN, for the launch that joins the parts
      if (32 * w + c < rows) {
        const long long part = (2LL * blockIdx.x + (blk0 == 0 ? 1 : 0)) * R + 32 * w + c;
        const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
        if (!whole && hh == 0) a.part_ml[part] = make_float2(m - kLift<F16>, sum);
#pragma unroll
        for (int db = 0; db < ND; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int dim = 32 * db + 8 * q + 4 * hh;
            ta_f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = far ? NAN : sum == 0.f ? 0.f : o[db][4 * q + e] * inv;
            if (whole) {
              ta_u32x2 z;
              z.x = narrow<F16>(v[0]) | static_cast<unsigned>(narrow<F16>(v[1])) << 16;
              z.y = narrow<F16>(v[2]) | static_cast<unsigned>(narrow<F16>(v[3])) << 16;
              *reinterpret_cast<ta_u32x2*>(a.out + q_row * D + dim) = z;
            } else {
              *reinterpret_cast<ta_f32x4*>(a.part_o + part * D + dim) = v;
            }
          }
      }
      __syncthreads();  // the ring is free again
    }
    u += stop - in_tile;
    if (u < end && u == base + t.units) {
      base += t.units;
      do t = uniform_tiles_of<R, B>(a, ++s);
      while (t.units == 0);
    }
  }
}

// One workgroup per node and 4 heads, a wave for each row: joins the parts of
// rows whose keys were shared out, and does over the rows that came out
// infinite or NaN (or whose scores lie too far out: far_out), one key at a time
// and only the keys that have a weight (a product with a weight of zero lets what
// is not seen through).
template <int D, bool F16, int R, int B>
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
  if (!__builtin_amdgcn_ballot_w64(again)) return;

  const uint16_t* q = a.q + (static_cast<long long>(n) * a.H + h) * D;
  const int ps = 1 << a.page_shift;
  // the key and value of position or node j, null where the row does not see it
  auto key = [&](int j, const uint16_t*& v) -> const uint16_t* {
    if (j < t.len) {
      const int page = a.table[static_cast<long long>(s) * a.max_pages + (j >> a.page_shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_pages)) return nullptr;
      const long long at = ((static_cast<long long>(page) * a.Hkv + hk) * ps + (j & (ps - 1))) * D;
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
  auto score = [&](int j, const uint16_t*& v) {  // one key a lane; v null where it has no weight
    v = nullptr;
    const uint16_t* k = j < keys ? key(j, v) : nullptr;
    if (!k) return -INFINITY;
    float x = 0.f;
    for (int d = 0; d < D; ++d) x += widen<F16>(q[d]) * widen<F16>(k[d]);
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
          const float x = widen<F16>(reinterpret_cast<const uint16_t*>(vi)[lane * E + e]);
          // a weight too small for fp32 is still not zero: an infinity stays one
          o[e] += (__builtin_isinf(x) ? fmaxf(pi, 1.17549435e-38f) : pi) * x;
        }
      }
    }
  for (int e = 0; e < E; ++e) out[lane * E + e] = narrow<F16>(sum != sum ? NAN : o[e]);
}

// Workgroups that fit the 256 CUs at once, by LDS (a ring takes 64 KiB with
// head_dim 64 and 128 KiB with 128) and, in the kernel of many rows, by registers.
constexpr int resident(int D, int R) { return R == 128 ? (D == 64 ? 768 : 512) : (D == 64 ? 512 : 256); }

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

int workgroups_of(int n_heads, int n_kv_heads, int head_dim, int num_seqs, int max_nodes, int max_pages, int page_size) {
  return static_cast<int>(std::min<long long>(most_units(n_heads, n_kv_heads, num_seqs, max_nodes, max_pages, page_size), resident(head_dim, rows_of_tile(n_heads, n_kv_heads, max_nodes))));
}

template <int D, bool F16, int RT>
void launch_tree(const TreeArgs& a, hipStream_t s) {
  IRON_LAUNCH((tree_attention_kernel<D, F16, RT>), dim3(a.workgroups), dim3(256), 0, s, a);
  IRON_LAUNCH((tree_join_kernel<D, F16, 16 * RT, kBlock>), dim3(a.num_nodes, (a.H + 3) / 4), dim3(256), 0, s, a);
}

template <int D, bool F16>
void launch_rows(const TreeArgs& a, int R, hipStream_t s) {
  if (R == 16)
    launch_tree<D, F16, 1>(a, s);
  else if (R == 32)
    launch_tree<D, F16, 2>(a, s);
  else {
    IRON_LAUNCH((tree_wide_kernel<D, F16>), dim3(a.workgroups), dim3(256), 0, s, a);
    IRON_LAUNCH((tree_join_kernel<D, F16, 128, kWideBlock>), dim3(a.num_nodes, (a.H + 3) / 4), dim3(256), 0, s, a);
  }
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

}  // namespace
}  // namespace iron

using namespace iron;

extern "C" long long iron_tree_attention_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int num_seqs,
                                                         int num_nodes, int max_nodes, int max_pages, int page_size) {
  if (check_shape(n_heads, n_kv_heads, head_dim, num_seqs, num_nodes, max_nodes, max_pages, page_size)) return -1;
  const long long slots = 2LL * workgroups_of(n_heads, n_kv_heads, head_dim, num_seqs, max_nodes, max_pages, page_size) *
                          rows_of_tile(n_heads, n_kv_heads, max_nodes);
  return slots * head_dim * 4 + slots * 8 + (num_seqs + 1 + num_nodes) * 4LL;
}

extern "C" int iron_tree_attention(const void* q, const void* k_new, const void* v_new, const void* k_pages,
                                   const void* v_pages, const int* page_table, const int* seq_lens,
                                   const int* node_starts, const int* tree_mask, void* out, int dtype, int n_heads,
                                   int n_kv_heads, int head_dim, int num_pages, int page_size, int num_seqs,
                                   int max_pages, int num_nodes, int max_nodes, float scale, void* workspace,
                                   long long workspace_bytes, void* stream) {
  const char* who = "iron_tree_attention";
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
  const long long need = iron_tree_attention_workspace_bytes(n_heads, n_kv_heads, head_dim, num_seqs, num_nodes,
                                                             max_nodes, max_pages, page_size);
  IRON_REQUIRE(workspace && aligned16(workspace), "%s: the workspace must be given and 16-byte aligned", who);
  IRON_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes, %lld needed", who, workspace_bytes, need);
  TreeArgs a;
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
  a.workgroups = workgroups_of(n_heads, n_kv_heads, head_dim, num_seqs, max_nodes, max_pages, page_size);
  const long long slots = 2LL * a.workgroups * R;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * head_dim);
  a.prefix = reinterpret_cast<int*>(a.part_ml + slots);
  a.owner = a.prefix + num_seqs + 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64)
    dtype ? launch_rows<64, true>(a, R, s) : launch_rows<64, false>(a, R, s);
  else
    dtype ? launch_rows<128, true>(a, R, s) : launch_rows<128, false>(a, R, s);
  return check_launch("tree_attention");
}
