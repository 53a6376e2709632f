// Attention of drafted trees over a paged KV cache of 4-bit rows (int4_rows.hpp):
// tree_attention.hip's mathematics, tiles and shares of work; the cached keys and
// values are b + s (16 + code), the tree's own are 16-bit rows.
//
// Roundings: in bf16 calls, cached keys, values and weights are rounded once to fp16,
// an eighth of the result's own rounding each (the whole error 1.01-1.08 times that of
// one rounding, root mean squares). In fp16 calls that would be 2.7 times; there keys
// are not rounded (s in two parts, b by a product of its own:
// S = K_high Q + K_low Q + b sum(q)) and weights go in two parts: 1.31-1.43 times.
//
// Measured (32 / 8 heads; a large copy moves 4.84 TB/s, a large library product does
// 1.28-1.39 PFLOP/s): 64 sequences of 150-16384 positions, one token each, head_dim 64:
// 48 us, the kernel 43 for 182 MB (with a 16-bit cache 94). One token behind 2047: 8.5 us
// in a graph. 8 trees of 26 nodes behind 37-3968: 21 us. 2 trees of 64 nodes behind 20011
// and 32768, head_dim 128, fp16: 143 us, 400 TFLOP/s of the mathematics' own products.
#include "tree_common.hpp"

namespace iron {
namespace {

// A wave's loads of a block: its 16 keys' codes and pairs, K's and V's. Lane
// (key c, quad) has quarter `quad` of key c's row.
template <int D>
struct Quarter {
  unsigned codes[D / 32];
  unsigned pair;
};

// Buffer loads: the rows' address is the wave's, in scalar registers, a lane's offset
// the same for all blocks (as global loads, each had its address computed in 64 bits).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const unsigned char* rows) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(rows), 0, 0x7fffffff, kBufferFlags);
}
template <int D>
__device__ __forceinline__ Quarter<D> load_quarter(const unsigned char* rows, unsigned at_codes, unsigned at_pair) {
  const __amdgpu_buffer_rsrc_t rsrc = rows_at(rows);
  Quarter<D> x;
  if constexpr (D == 64) {
    const ta_u32x2 v = __builtin_bit_cast(ta_u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at_codes, 0, 0));
    x.codes[0] = v.x, x.codes[1] = v.y;
  } else {
    const ta_u32x4 v = __builtin_bit_cast(ta_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at_codes, 0, 0));
    x.codes[0] = v.x, x.codes[1] = v.y, x.codes[2] = v.z, x.codes[3] = v.w;
  }
  x.pair = __builtin_amdgcn_raw_buffer_load_b32(rsrc, at_pair, 0, 0);
  return x;
}

// The largest of three numbers; the compiler's own makes quiet NaN of its operands first,
// at an instruction each. It does not see that this reads a product's result, which takes
// 11 (16x16) or 19 (32x32) wait states: products go through settle() first.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

template <int RT>
__device__ __forceinline__ void settle(ta_f32x4 (&a)[2][RT]) {
  if constexpr (RT == 1)
    asm volatile("s_nop 10" : "+v"(a[0][0]), "+v"(a[1][0]));
  else
    asm volatile("s_nop 10" : "+v"(a[0][0]), "+v"(a[1][0]), "+v"(a[0][1]), "+v"(a[1][1]));
}
__device__ __forceinline__ void settle(ta_f32x16& a) { asm volatile("s_nop 15\n\ts_nop 2" : "+v"(a)); }

// Eight values of a quarter (word kk) as the fp16 operand of a product.
template <int D>
__device__ __forceinline__ ta_u32x4 unpack(const Quarter<D>& x, int kk) {
  unsigned w[4];
  int4_unpack8(x.codes[kk], int4_scale(x.pair), int4_base(x.pair), w);
  return ta_u32x4{w[0], w[1], w[2], w[3]};
}

// The same without rounding: half a value is high + low + b / 2 (int4_split8).
template <int D>
__device__ __forceinline__ void unpack(const Quarter<D>& x, int kk, ta_u32x4& high, ta_u32x4& low) {
  const i4_f16x2 s = int4_scale(x.pair), s_high = int4_scale(x.pair & 0xffe0u);
  unsigned a[4], b[4];
  int4_split8(x.codes[kk], s_high, s - s_high, a, b);
  high = ta_u32x4{a[0], a[1], a[2], a[3]};
  low = ta_u32x4{b[0], b[1], b[2], b[3]};
}

// A number as two fp16 ones, the upper in the low half.
__device__ __forceinline__ unsigned split_fp16(float x) {
  const _Float16 high = static_cast<_Float16>(x), low = static_cast<_Float16>(x - static_cast<float>(high));
  return __builtin_bit_cast(unsigned, ta_f16x2{high, low});
}

// A row of q as the fp16 operand beside cached keys, scaled by a power of two; the
// scores get the inverse (factor). bf16: the largest element comes into [2^14, 2^15), so
// that none is cut and those of 2^-29 of it and more stay exact. fp16: into [2^9, 2^10),
// but by 2^24 at most, so that the sums of a quarter (32 elements at most), which b is
// multiplied by, fit fp16 in two parts, those of subnormal rows too; elements of 2^-23 of
// the largest and more stay exact.
// A row with an infinity or NaN comes out with one, and is done over by the join.
template <bool F16, bool WIDE, int NK>
__device__ __forceinline__ float to_fp16(ta_u32x4 (&q)[NK], float scale) {
  float top = 0.f;
  if constexpr (F16) {
    ta_f16x2 most = {0, 0};
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(ta_f16x2, q[kk][i] & 0x7fff7fffu));
    top = fmaxf(static_cast<float>(most[0]), static_cast<float>(most[1]));
  } else {
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(lo_bf16(q[kk][i])), fabsf(hi_bf16(q[kk][i]))));
  }
  if constexpr (WIDE) {  // two lanes have a row, or four
    float x, y;
    swap32(top, x, y);
    top = fmaxf(x, y);
  } else {
    top = row_max(top);
  }
  int e = (F16 ? 10 : 15) - __builtin_amdgcn_frexp_expf(top);
  if constexpr (F16) {  // in two steps that fp16 has
    e = min(e, 24);
    const _Float16 a = static_cast<_Float16>(__builtin_amdgcn_ldexpf(1.f, e >> 1)), b = static_cast<_Float16>(__builtin_amdgcn_ldexpf(1.f, e - (e >> 1)));
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned x = q[kk][i];  // a bit cast of the vector's element itself takes its first one
        q[kk][i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(ta_f16x2, x) * ta_f16x2{a, a} * ta_f16x2{b, b});
      }
  } else {
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[kk][i] = pack2<true>(__builtin_amdgcn_ldexpf(lo_bf16(q[kk][i]), e), __builtin_amdgcn_ldexpf(hi_bf16(q[kk][i]), e));
  }
  const float factor = __builtin_amdgcn_ldexpf(scale, -e);
  return factor == INFINITY ? NAN : factor;  // done over, too
}

// Workgroups of the kernels of few and of many rows that fit the 256 CUs at once, by
// their registers.
constexpr int few_resident(int D, int RT, bool F16) { return D == 64 ? (RT == 1 ? 1024 : 768) : RT == 1 && !F16 ? 768 : 512; }
constexpr int wide_resident(int D, bool F16) { return D == 64 && !F16 ? 768 : 512; }

// Few rows: a tile of 16 RT rows, a workgroup of 4 waves. Wave w has keys 16 w ..
// + 15 of each block of 64 and all rows, so that nothing is shared until the end.
// A lane has a quarter of a key's row, which it loads (a step ahead, into registers)
// and dequantizes itself. K's quarters are the A operand of S^T = K Q^T as
// they stand, with Q's dims in the same order; V's go through the wave's own LDS,
// 16-bit rows in, V^T out by transposed reads. Two blocks make a step: the weights of
// 2 x 4 keys, rounded to fp16, are the 8 elements of the B operand of O^T += V^T P^T.
// Bound by memory, half of the waves' time waiting for it, at four waves to a SIMD: 2, 4,
// 6 and 8 blocks ahead took 51, 55-61, 74 and 70 us for the batch above (registers, code).
template <int D, bool F16, int RT>
__global__ __launch_bounds__(256, few_resident(D, RT, F16) / 256) void tree4_kernel(TreeArgs a) {
  constexpr int R = 16 * RT, B = kBlock, kRow = kInt4Row<D>, kWide = D * 2;
  constexpr int NK = D / 32, ND = D / 16;
  constexpr int kOwn = 32 * kWide > R * D * 4 ? 32 * kWide : R * D * 4;  // LDS of a wave: V of two blocks, at the end its output
  __shared__ __attribute__((aligned(16))) unsigned char lds[4 * kOwn];
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
  unsigned char* own = lds + w * kOwn;
  const unsigned at_codes = c * kRow + quad * (D / 8), at_pair = c * kRow + D / 2 + quad * 4;
  const int trow = 4 * quad + (c >> 2), tcol = 4 * (c & 3);  // this lane's address of a transposed V read
  const unsigned char* k_pages = reinterpret_cast<const unsigned char*>(a.k_pages);
  const unsigned char* v_pages = reinterpret_cast<const unsigned char*>(a.v_pages);

  // V rows of 16 keys: this lane's quarter in, four keys of dims 16 dt + c out.
  auto put_v = [&](int half, int kk, ta_u32x4 x) {
    *reinterpret_cast<ta_u32x4*>(own + half * 16 * kWide + c * kWide + v_slot<D>(c, quad * NK + kk) * 16) = x;
  };
  auto get_v = [&](int half, int dt) {
    const int dim = 16 * dt + tcol;
    return __builtin_bit_cast(ta_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ta_i16x4*)(
        own + half * 16 * kWide + trow * kWide + v_slot<D>(trow, dim >> 3) * 16 + (dim & 7) * 2)));
  };
  // bits of V^T's four keys that count: of `valid` keys
  auto keep01 = [&](int valid) { return (4 * quad < valid ? 0xffffu : 0u) | (4 * quad + 1 < valid ? 0xffff0000u : 0u); };
  auto keep23 = [&](int valid) { return (4 * quad + 2 < valid ? 0xffffu : 0u) | (4 * quad + 3 < valid ? 0xffff0000u : 0u); };

  while (u < end) {
    const int tu = t.tile_units(), tile = uniform((u - base) / tu), in_tile = (u - base) - tile * tu;
    const int stop = min(tu, in_tile + (end - u)), blk0 = max(in_tile - kOver, 0), n = stop - kOver - blk0;
    const int hk = uniform(tile / t.row_tiles), row0 = (tile - hk * t.row_tiles) * R;
    const int rows = min(R, t.nodes * G - row0);
    if (n > 0) {
      if (hk == 0 && blk0 == 0)  // for the launch that joins the parts
        for (int i = row0 / G + tid; i <= (row0 + rows - 1) / G; i += 256) a.owner[t.first + i] = s;
      const int* table = a.table + static_cast<long long>(s) * a.max_pages;
      const int cached = min(n, t.cached - blk0);  // blocks of this part that are the cache's (the rest are the tree's)
      const long long head = static_cast<long long>(hk) * ps * kRow, page_bytes = static_cast<long long>(a.Hkv) * ps * kRow;

      // A block of the cache: where this wave's keys lie, and how many of them count.
      auto page_of = [&](int i) { return uniform_word(table, min((blk0 + min(i, cached - 1)) * B + 16 * w, t.len - 1) >> a.page_shift); };
      auto rows_of = [&](int i, int page) {
        const bool real = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages);
        return (real ? page : 0) * page_bytes + head + (((blk0 + min(i, cached - 1)) * B + 16 * w) & (ps - 1)) * kRow;
      };
      auto valid_of = [&](int i, int page) {
        const bool real = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages);
        return real && i < cached ? max(min(t.len - ((blk0 + i) * B + 16 * w), 16), 0) : 0;
      };
      // The two blocks of a step, loaded while the step before it is worked on; their
      // pages are read a step earlier still.
      Quarter<D> kq[2], vq[2];
      int valid[2], page[2] = {0, 0};
      auto read_pages = [&](int i) {
        page[0] = page_of(i);
        page[1] = page_of(i + 1);
      };
      auto issue = [&](int i) {  // blocks i and i + 1 (behind the last one: that one again, of which nothing counts)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const long long at = rows_of(i + j, page[j]);
          valid[j] = valid_of(i + j, page[j]);
          kq[j] = load_quarter<D>(k_pages + at, at_codes, at_pair);
          vq[j] = load_quarter<D>(v_pages + at, at_codes, at_pair);
        }
        read_pages(i + 2);
      };
      if (cached > 0) {
        read_pages(0);
        issue(0);
      }
      // Q: the B operand of S^T = K Q^T (column: row 16 rt + c; dims D / 4 quad + 8 kk .. + 8)
      ta_u32x4 qf[RT][NK];
      int node[RT];
      ta_f32x4 o[RT][ND];
      float m[RT], off[RT], l[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = min(row0 + 16 * rt + c, t.nodes * G - 1), in_tree = r / G;
        node[rt] = t.first + in_tree;
        const uint16_t* qp = a.q + (static_cast<long long>(node[rt]) * a.H + hk * G + (r - in_tree * G)) * D + quad * (D / 4);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[rt][kk] = *reinterpret_cast<const ta_u32x4*>(qp + 8 * kk);
        m[rt] = -INFINITY;
        off[rt] = l[rt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[rt][dt] = ta_f32x4{0.f, 0.f, 0.f, 0.f};
      }

      // Softmax in the log2 domain, p = 2^(s c - m). The row's maximum m moves only
      // when a score passes it by more than 8, so p <= 2^8 and O is rarely
      // rescaled; sum(p v) / sum(p) does not depend on which m is used.
      auto raise = [&](const float (&top)[RT]) {  // of the lane's scores, times c
        bool grow = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) grow |= top[rt] > m[rt] + 8.f;
        if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const float all = row_max(top[rt]);
            if (all > m[rt] + 8.f) {
              const float alpha = __builtin_amdgcn_exp2f(m[rt] - all);  // 0 from m = -inf
              m[rt] = all;
              off[rt] = all - kLift<true>;
              l[rt] *= alpha;
#pragma unroll
              for (int dt = 0; dt < ND; ++dt) o[rt][dt] *= alpha;
            }
          }
        }
      };
      // The tree's own keys first, while the cache's are on their way: 16-bit rows, weights
      // in two parts (split4), V^T's 4 keys given twice.
      for (int i = max(cached, 0); i < n; ++i) {
        const int j0 = (blk0 + i - t.cached) * B + 16 * w, have = min(t.nodes - j0, 16);
        if (have <= 0) continue;
        const long long key = (static_cast<long long>(t.first + min(j0 + c, t.nodes - 1)) * a.Hkv + hk) * D + quad * (D / 4);
        ta_f32x4 sc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt] = ta_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const ta_u32x4 kf = *reinterpret_cast<const ta_u32x4*>(a.k_new + key + 8 * kk);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt] = mfma<F16>(kf, qf[rt][kk], sc[rt]);
          put_v(0, kk, *reinterpret_cast<const ta_u32x4*>(a.v_new + key + 8 * kk));
        }
        asm volatile("" ::: "memory");
        float top[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int word = a.mask[static_cast<long long>(node[rt]) * a.words + (j0 >> 5)] >> ((j0 & 31) + 4 * quad);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[rt][e] = 4 * quad + e < have && (word >> e & 1) ? sc[rt][e] : -INFINITY;
          top[rt] = fmaxf(fmaxf(sc[rt][0], sc[rt][1]), fmaxf(sc[rt][2], sc[rt][3])) * a.scale_log2;
        }
        raise(top);
        const unsigned m01 = keep01(have), m23 = keep23(have);
        ta_u32x4 pf[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[rt][e], a.scale_log2, -off[rt]));
          l[rt] += (p[0] + p[1]) + (p[2] + p[3]);
          pf[rt] = split4<F16>(p);
        }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          ta_u32x2 vt = get_v(0, dt);
          vt.x &= m01;
          vt.y &= m23;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma<F16>(ta_u32x4{vt.x, vt.y, vt.x, vt.y}, pf[rt], o[rt][dt]);
        }
        asm volatile("" ::: "memory");
      }

      float cs[RT];
      unsigned q_half[RT];  // fp16: half the sum of the lane's dims, in two parts, b's factor
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        cs[rt] = to_fp16<F16, false>(qf[rt], a.scale_log2);
        if constexpr (F16) {
          float sum = 0.f;
#pragma unroll
          for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = add2<true>(qf[rt][kk][i], sum);
          q_half[rt] = split_fp16(sum * 0.5f);
          cs[rt] *= 2.f;
        }
      }
      auto step = [&] {
        if (valid[0] + valid[1] == 0) return;
        ta_f32x4 sc[2][RT];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) put_v(b, kk, unpack<D>(vq[b], kk));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[b][rt] = ta_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) {
            if constexpr (F16) {
              ta_u32x4 high, low;
              unpack<D>(kq[b], kk, high, low);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) sc[b][rt] = mfma<true>(low, qf[rt][kk], mfma<true>(high, qf[rt][kk], sc[b][rt]));
            } else {
              const ta_u32x4 kf = unpack<D>(kq[b], kk);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) sc[b][rt] = mfma<true>(kf, qf[rt][kk], sc[b][rt]);
            }
          }
          if constexpr (F16) {  // b, twice, times the two parts of the sum of the quarter's dims
            const unsigned bb = __builtin_bit_cast(unsigned, int4_base(kq[b].pair));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[b][rt] = mfma<true>(ta_u32x4{bb, 0, 0, 0}, ta_u32x4{q_half[rt], 0, 0, 0}, sc[b][rt]);
          }
        }
        asm volatile("" ::: "memory");
        settle(sc);
        const bool some = valid[0] + valid[1] < 32;  // keys that are none: no score, and values that cannot do harm
        if (some) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) sc[b][rt][e] = 4 * quad + e < valid[b] ? sc[b][rt][e] : -INFINITY;
        }
        ta_u32x2 vt[2][ND];
        auto get = [&](int b) {
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) vt[b][dt] = get_v(b, dt);
          if (some) {
            const unsigned m01 = keep01(valid[b]), m23 = keep23(valid[b]);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
              vt[b][dt].x &= m01;
              vt[b][dt].y &= m23;
            }
          }
        };
        if constexpr (!F16) {
          get(0);
          get(1);
        }
        float top[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const ta_f32x4 x = sc[0][rt], y = sc[1][rt];
          top[rt] = max3(max3(max3(x[0], x[1], x[2]), x[3], y[0]), max3(y[1], y[2], y[3]), y[3]) * cs[rt];
        }
        raise(top);
        if constexpr (F16) {  // weights in two parts (split4), V^T's 4 keys given twice
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            get(b);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              float p[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[b][rt][e], cs[rt], -off[rt]));
              l[rt] += (p[0] + p[1]) + (p[2] + p[3]);
              const ta_u32x4 pf = split4<true>(p);
#pragma unroll
              for (int dt = 0; dt < ND; ++dt) o[rt][dt] = mfma<true>(ta_u32x4{vt[b][dt].x, vt[b][dt].y, vt[b][dt].x, vt[b][dt].y}, pf, o[rt][dt]);
            }
            asm volatile("" ::: "memory");
          }
        } else {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            ta_u32x4 pf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const ta_f32x4 x = sc[i >> 1][rt];
              pf[i] = pack2<true>(__builtin_amdgcn_exp2f(fmaf(x[2 * (i & 1)], cs[rt], -off[rt])), __builtin_amdgcn_exp2f(fmaf(x[2 * (i & 1) + 1], cs[rt], -off[rt])));
              l[rt] = add2<true>(pf[i], l[rt]);
            }
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[rt][dt] = mfma<true>(ta_u32x4{vt[0][dt].x, vt[0][dt].y, vt[1][dt].x, vt[1][dt].y}, pf, o[rt][dt]);
          }
        }
        asm volatile("" ::: "memory");
      };
      for (int i = 0; i < cached; i += 2) {
        step();
        issue(i + 2);
      }

      // The four waves' parts of the tile meet in LDS.
      const bool whole = n == t.blocks;
      const long long slot = 2LL * blockIdx.x + (blk0 == 0 ? 1 : 0);
      float* mine_o = reinterpret_cast<float*>(own);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = 16 * rt + c;
        const float sum = row_sum(l[rt]);
        if (quad == 0) {
          stat_m[w][r] = m[rt] - kLift<true>;
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
          const ta_f32x4 part = f * *reinterpret_cast<const ta_f32x4*>(reinterpret_cast<const float*>(lds + i * kOwn) + r * D + ((c4 ^ (r & 15)) * 4));
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
      __syncthreads();  // the waves' LDS is free again
    }
    u += stop - in_tile;
    if (u < end && u == base + t.units) {
      base += t.units;
      do t = uniform_tiles_of<R, B>(a, ++s);
      while (t.units == 0);
    }
  }
}

// Many rows: a tile of 128 rows, a workgroup of 4 waves with 32 rows each. The waves
// dequantize blocks of 32 keys together (8 rows of K and of V each) into a ring of
// 16-bit rows in LDS, two blocks ahead of their use and four ahead of it into
// registers; a block is dequantized once for 128 rows. From there on it is
// tree_wide_kernel: scores of the next block among this one's softmax, one barrier a
// block. The cache's blocks come first, with fp16 products, then the tree's, with
// those of its type; a row's maximum, sum and output go on through both.
template <int D, bool F16>
__global__ __launch_bounds__(256, wide_resident(D, F16) / 256) void tree4_wide_kernel(TreeArgs a) {
  constexpr int R = 128, B = kWideBlock, kRow = D * 2, kHalf = B * kRow, kRing = 3;
  constexpr int kStage = F16 ? 3 * kHalf : 2 * kHalf;  // K, V and, with fp16, K's lower parts; b's behind the ring
  constexpr int kRow4 = kInt4Row<D>, NW = D / 64;  // words of codes (16-byte chunks of 16-bit rows) of a lane and block
  constexpr int NK = D / 16, ND = D / 32;
  __shared__ __attribute__((aligned(16))) unsigned char ring[kRing * kStage + (F16 ? kRing * B * 16 : 0)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  const int G = a.G, ps = 1 << a.page_shift;
  Share sh;
  if (!share_of<R, B>(a, blockIdx.x, sh)) return;
  int u = sh.at, s = sh.s, base = sh.base;
  const int end = sh.end;
  Tiles t = sh.t;

  // This lane's part of a block: NW chunks from chunk0 on of row srow.
  const int srow = 8 * w + (lane >> 3), chunk0 = NW * (lane & 7);
  const unsigned at_codes = (lane >> 3) * kRow4 + chunk0 * 4, at_pair = (lane >> 3) * kRow4 + D / 2 + (lane & 7) / 2 * 4;
  const unsigned k_store = srow * kRow + k_slot<D>(srow & 15, chunk0) * 16, v_store = kHalf + srow * kRow + wide_v_slot<D>(srow, chunk0) * 16;
  const int trow = 4 * hh + ((lane & 15) >> 2), tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  // Both swizzles are exclusive ors, so a fragment's address is the first one's with
  // the fragment's own bits turned: one register for each operand.
  const unsigned k_first = c * kRow + k_slot<D>(c & 15, hh) * 16;
  const unsigned v_first = kHalf + trow * kRow + wide_v_slot<D>(trow, tcol >> 3) * 16 + (tcol & 7) * 2;
  const unsigned char* k_pages = reinterpret_cast<const unsigned char*>(a.k_pages);
  const unsigned char* v_pages = reinterpret_cast<const unsigned char*>(a.v_pages);

  while (u < end) {
    const int tu = t.tile_units(), tile = uniform((u - base) / tu), in_tile = (u - base) - tile * tu;
    const int stop = min(tu, in_tile + (end - u)), blk0 = max(in_tile - kOver, 0), n = stop - kOver - blk0;
    const int hk = uniform(tile / t.row_tiles), row0 = (tile - hk * t.row_tiles) * R;
    const int rows = min(R, t.nodes * G - row0);
    if (n > 0) {
      if (hk == 0 && blk0 == 0)  // for the launch that joins the parts
        for (int i = row0 / G + tid; i <= (row0 + rows - 1) / G; i += 256) a.owner[t.first + i] = s;
      const int r = min(row0 + 32 * w + c, t.nodes * G - 1), in_tree = r / G;
      const int node = t.first + in_tree;
      const long long q_row = static_cast<long long>(node) * a.H + hk * G + (r - in_tree * G);
      ta_f32x16 o[ND];
      float m = -INFINITY, off = 0.f, l = 0.f;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[db][j] = 0.f;
      const bool idle = 32 * w >= rows;  // none of the wave's rows is one

      // Blocks blk0 .. of the cache (CACHE) or of the tree.
      auto phase = [&](auto cache) {
        constexpr bool CACHE = decltype(cache)::value, T16 = CACHE || F16, EXACT = CACHE && F16;  // T16: fp16 operands
        constexpr bool ONE = EXACT || (!CACHE && D == 128);  // K's fragments one ahead, not all at once: what registers there are
        const int nb = CACHE ? min(n, t.cached - blk0) : n - max(min(n, t.cached - blk0), 0);
        if (nb <= 0) return;
        const int first = CACHE ? blk0 : max(blk0 - t.cached, 0), have = CACHE ? t.len : t.nodes;
        const int whole_blocks = have / B - first;  // the first ones of them, with no key behind the last
        // Q: the B operand of S^T = K Q^T (column: row 32 w + c; dims 16 kk + 8 hh .. + 8)
        ta_u32x4 qf[NK];
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[kk] = *reinterpret_cast<const ta_u32x4*>(a.q + q_row * D + 16 * kk + 8 * hh);
        float cs = CACHE ? to_fp16<F16, true>(qf, a.scale_log2) : a.scale_log2;
        ta_u32x4 q_half = {0, 0, 0, 0};  // half the sums of the quarters' dims, each in two parts: b's factors (the upper lanes' are 0)
        if constexpr (EXACT) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float sum = 0.f, x, y;
#pragma unroll
            for (int kk = g * NK / 4; kk < (g + 1) * NK / 4; ++kk)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum = add2<true>(qf[kk][i], sum);
            swap32(sum, x, y);
            q_half[g] = hh ? 0 : split_fp16((x + y) * 0.5f);
          }
          cs *= 2.f;
        }

        // A block's rows on their way: codes and pairs, or 16-bit chunks.
        struct Ahead {
          ta_u32x4 k[CACHE ? 1 : NW], v[CACHE ? 1 : NW];
          unsigned kp, vp;
        };
        constexpr int kDeep = D == 128 && (EXACT || !CACHE) ? 1 : 2;  // blocks on their way: what registers there are
        Ahead ahead[2];
        unsigned holes = 0;  // bits 2 (i % 8) and + 1: the two pages of block i's 16 rows each are none
        const int* table = a.table + static_cast<long long>(s) * a.max_pages;
        const long long head = static_cast<long long>(hk) * ps * kRow4, page_bytes = static_cast<long long>(a.Hkv) * ps * kRow4;
        int page0 = 0, page1 = 0;
        auto pages_of = [&](int i) {
          if constexpr (CACHE) {
            const int pos = (first + min(i, nb - 1)) * B;
            page0 = uniform_word(table, pos >> a.page_shift);
            page1 = uniform_word(table, min(pos + 16, t.len - 1) >> a.page_shift);
          }
        };
        auto issue = [&](int i, Ahead& x) {  // block i, or the last one again
          const int blk = first + min(i, nb - 1);
          if constexpr (CACHE) {
            const bool none0 = static_cast<unsigned>(page0) >= static_cast<unsigned>(a.num_pages);
            const bool none1 = static_cast<unsigned>(page1) >= static_cast<unsigned>(a.num_pages);
            holes = (holes & ~(3u << (2 * (i & 7)))) | ((none0 ? 1u : 0u) | (none1 ? 2u : 0u)) << (2 * (i & 7));
            const int page = w < 2 ? (none0 ? 0 : page0) : (none1 ? 0 : page1);
            const long long at = page * page_bytes + head + ((blk * B + 8 * w) & (ps - 1)) * kRow4;
            if constexpr (NW == 1) {
              x.k[0].x = *reinterpret_cast<const unsigned*>(k_pages + at + at_codes);
              x.v[0].x = *reinterpret_cast<const unsigned*>(v_pages + at + at_codes);
            } else {
              const ta_u32x2 k = *reinterpret_cast<const ta_u32x2*>(k_pages + at + at_codes), v = *reinterpret_cast<const ta_u32x2*>(v_pages + at + at_codes);
              x.k[0].x = k.x, x.k[0].y = k.y, x.v[0].x = v.x, x.v[0].y = v.y;
            }
            x.kp = *reinterpret_cast<const unsigned*>(k_pages + at + at_pair);
            x.vp = *reinterpret_cast<const unsigned*>(v_pages + at + at_pair);
            pages_of(i + 1);
          } else {
            const long long at = (static_cast<long long>(t.first + min(blk * B + srow, t.nodes - 1)) * a.Hkv + hk) * D + chunk0 * 8;
#pragma unroll
            for (int e = 0; e < NW; ++e) {
              x.k[e] = *reinterpret_cast<const ta_u32x4*>(a.k_new + at + 8 * e);
              x.v[e] = *reinterpret_cast<const ta_u32x4*>(a.v_new + at + 8 * e);
            }
          }
        };
        // Block i's rows into their stage; values of keys that are none become zeros, which cannot do harm.
        auto stage = [&](int i, const Ahead& x) {
          unsigned char* st = ring + i % kRing * kStage;
          const unsigned none = holes >> (2 * (i & 7)) & 3u;
          const bool gone = (i >= whole_blocks && (first + i) * B + srow >= have) || (none >> (w >> 1) & 1);
#pragma unroll
          for (int e = 0; e < NW; ++e) {
            ta_u32x4 k, v;
            if constexpr (CACHE) {
              unsigned y[4];
              if constexpr (EXACT) {
                const i4_f16x2 sk = int4_scale(x.kp), s_high = int4_scale(x.kp & 0xffe0u);
                unsigned z[4];
                int4_split8(e ? x.k[0].y : x.k[0].x, s_high, sk - s_high, y, z);
                *reinterpret_cast<ta_u32x4*>(st + 2 * kHalf + (k_store ^ 16 * e)) = ta_u32x4{z[0], z[1], z[2], z[3]};
                if (e == 0 && !(lane & 1)) *reinterpret_cast<unsigned*>(ring + kRing * kStage + i % kRing * B * 16 + srow * 16 + (lane & 7) * 2) = __builtin_bit_cast(unsigned, int4_base(x.kp));
              } else {
                int4_unpack8(e ? x.k[0].y : x.k[0].x, int4_scale(x.kp), int4_base(x.kp), y);
              }
              k = ta_u32x4{y[0], y[1], y[2], y[3]};
              int4_unpack8(e ? x.v[0].y : x.v[0].x, int4_scale(x.vp), int4_base(x.vp), y);
              v = ta_u32x4{y[0], y[1], y[2], y[3]};
            } else {
              k = x.k[e], v = x.v[e];
            }
            if (gone) v = ta_u32x4{0, 0, 0, 0};
            *reinterpret_cast<ta_u32x4*>(st + (k_store ^ 16 * e)) = k;
            *reinterpret_cast<ta_u32x4*>(st + (v_store ^ 16 * e)) = v;
          }
        };
        auto k_frag = [&](int i, int kk) {
          return *reinterpret_cast<const ta_u32x4*>(ring + ((i % kRing * kStage + k_first) ^ (32 * kk)));
        };
        auto low_frag = [&](int i, int kk) {
          return *reinterpret_cast<const ta_u32x4*>(ring + ((i % kRing * kStage + 2 * kHalf + k_first) ^ (32 * kk)));
        };
        auto base_frag = [&](int i) { return *reinterpret_cast<const ta_u32x4*>(ring + kRing * kStage + i % kRing * B * 16 + c * 16); };
        // V^T of keys 8 q + 4 hh .. + 3 of block i, dims 32 db + lane % 32
        auto v_frag = [&](int i, int q, int db) {
          return __builtin_bit_cast(ta_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ta_i16x4*)(
              ring + ((i % kRing * kStage + v_first) ^ (64 * db)) + 8 * q * kRow)));
        };
        // The row's maximum, when scores pass it by more than 8 (in the log2 domain; cf. tree4_kernel).
        auto raise = [&](ta_f32x16& sc) {
          settle(sc);
          float mx = max3(sc[0], sc[1], sc[2]);
#pragma unroll
          for (int j = 3; j < 15; j += 2) mx = max3(mx, sc[j], sc[j + 1]);
          mx = max3(mx, sc[15], sc[15]);
          if (__builtin_amdgcn_ballot_w64(mx * cs > m + 8.f)) {
            float x, y;
            swap32(mx, x, y);
            const float top = fmaxf(x, y) * cs;
            if (top > m + 8.f) {
              const float alpha = __builtin_amdgcn_exp2f(m - top);  // 0 from m = -inf
              m = top;
              off = top - kLift<true>;
              l *= alpha;
#pragma unroll
              for (int db = 0; db < ND; ++db) o[db] *= alpha;
            }
          }
        };
        // Weights 2 g and 2 g + 1 of the lane in two parts (cf. split4), where the cached values are exact.
        auto weights2 = [&](const ta_f32x16& sc, int g, unsigned& low) {
          const float p = __builtin_amdgcn_exp2f(fmaf(sc[2 * g], cs, -off)), q = __builtin_amdgcn_exp2f(fmaf(sc[2 * g + 1], cs, -off));
          const auto x = __builtin_amdgcn_cvt_pkrtz(p, q);
          low = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(p - static_cast<float>(x[0]), q - static_cast<float>(x[1])));
          l += p + q;
          return __builtin_bit_cast(unsigned, x);
        };
        // Weights 2 g and 2 g + 1 of the lane, rounded to 16 bits as the second product takes them; l sums those.
        auto weights = [&](const ta_f32x16& sc, int g) {
          const unsigned p = pack2<T16>(__builtin_amdgcn_exp2f(fmaf(sc[2 * g], cs, -off)), __builtin_amdgcn_exp2f(fmaf(sc[2 * g + 1], cs, -off)));
          l = add2<T16>(p, l);
          return p;
        };
        // Block i from its scores S^T: sc[j] is key 8 (j / 4) + 4 hh + j % 4, row 32 w + c.
        auto step = [&](int i, ta_f32x16& sc, ta_f32x16& next) {
          const unsigned none = holes >> (2 * (i & 7)) & 3u;
          if (!CACHE || i >= whole_blocks || none) {  // some of its keys are none, or not for every row
            const int j0 = (first + i) * B, left = have - j0;
            unsigned seen = left >= 32 ? ~0u : (1u << left) - 1;  // those that there are
            seen &= ~((none & 1 ? 0xffffu : 0u) | (none & 2 ? 0xffff0000u : 0u));
            if (!CACHE) seen &= a.mask[static_cast<long long>(node) * a.words + (j0 >> 5)];
            seen >>= 4 * hh;
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[j] = seen >> (8 * (j >> 2) + (j & 3)) & 1 ? sc[j] : -INFINITY;
          }
          // K's fragments of block i + 1 (behind the last block: a stage that nothing writes, for scores that go unused)
          ta_u32x4 kf[NK], low[NK], bf;
          if constexpr (EXACT) bf = base_frag(i + 1);
          if constexpr (ONE) {
            kf[0] = k_frag(i + 1, 0);
          } else {
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) kf[kk] = k_frag(i + 1, kk);
          }
          raise(sc);
          // In eight groups, held in this order by the scheduling barriers (cf. tree_wide_kernel).
          ta_u32x4 pf[2], pl[2];  // P^T of keys 16 g + 4 hh .. + 3 and + 8 .. + 11, its lower part
          ta_u32x2 vt[4][ND];
          auto pv = [&](int g, int db) {
            const ta_u32x4 v = {vt[2 * g][db].x, vt[2 * g][db].y, vt[2 * g + 1][db].x, vt[2 * g + 1][db].y};
            o[db] = mfma32<T16>(v, pf[g], o[db]);
            if constexpr (EXACT) o[db] = mfma32<T16>(v, pl[g], o[db]);
          };
          next = ta_f32x16{};
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (ONE)
              if (g + 1 < NK) kf[g + 1] = k_frag(i + 1, g + 1);
            if constexpr (EXACT) {
              if (g < NK) low[g] = low_frag(i + 1, g);
              if (g == 0) next = mfma32<T16>(bf, q_half, next);
            }
            if (g < NK) next = mfma32<T16>(kf[g], qf[g], next);
            if constexpr (EXACT)
              if (g < NK) next = mfma32<T16>(low[g], qf[g], next);
            if (g >= 4 && g - 4 < ND) pv(0, g - 4);
#pragma unroll
            for (int e = g * ND / 2; e < (g + 1) * ND / 2; ++e) vt[e / ND][e % ND] = v_frag(i, e / ND, e % ND);
            if constexpr (EXACT) {
              unsigned x;
              pf[g / 4][g % 4] = weights2(sc, g, x);
              pl[g / 4][g % 4] = x;
            } else {
              pf[g / 4][g % 4] = weights(sc, g);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int db = 0; db < ND; ++db) pv(1, db);
        };
        auto meet = [&] {  // every wave's LDS accesses so far are done
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        };
        // Stages: i (V being read), i + 1 (K being read), i + 2 being written, which every wave has left.
        auto turn = [&](int i, ta_f32x16& sc, ta_f32x16& next, Ahead& x) {
          meet();  // block i + 1 is there, and block i - 1's stage read by all
          if (i + 2 < nb) stage(i + 2, x);
          issue(i + 2 + kDeep, x);
          if (!idle) step(i, sc, next);
        };
        pages_of(0);
        issue(0, ahead[0]);
        if (kDeep == 2) issue(1, ahead[1]);
        stage(0, ahead[0]);
        issue(kDeep, ahead[0]);
        if (nb > 1) stage(1, ahead[kDeep - 1]);
        issue(kDeep + 1, ahead[kDeep - 1]);
        meet();
        ta_f32x16 sa = {}, sb = {};
        if (!idle) {
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) {
            sa = mfma32<T16>(k_frag(0, kk), qf[kk], sa);
            if constexpr (EXACT) sa = mfma32<T16>(low_frag(0, kk), qf[kk], sa);
          }
          if constexpr (EXACT) sa = mfma32<T16>(base_frag(0), q_half, sa);
        }
        for (int i = 0; i < nb; i += 2) {
          turn(i, sa, sb, ahead[0]);
          if (i + 1 < nb) turn(i + 1, sb, sa, ahead[kDeep - 1]);
        }
        meet();  // the ring is free again
      };
      phase(std::true_type{});
      phase(std::false_type{});

      const bool whole = n == t.blocks;
      float l0, l1;
      swap32(l, l0, l1);
      const float sum = l0 + l1;
      const bool far = whole && far_out(m);  // NaN, for the launch that joins the parts
      if (32 * w + c < rows) {
        const long long part = (2LL * blockIdx.x + (blk0 == 0 ? 1 : 0)) * R + 32 * w + c;
        const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
        if (!whole && hh == 0) a.part_ml[part] = make_float2(m - kLift<true>, sum);
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

// Workgroups that fit the 256 CUs at once.
int resident(int D, int R) { return R < 128 ? few_resident(D, R / 16, false) : wide_resident(D, false); }

template <int D, bool F16, int RT>
void launch_few(TreeArgs a, hipStream_t s) {
  a.workgroups = std::min(a.workgroups, few_resident(D, RT, F16));
  IRON_LAUNCH((tree4_kernel<D, F16, RT>), dim3(a.workgroups), dim3(256), 0, s, a);
  IRON_LAUNCH((tree_join_kernel<D, F16, 16 * RT, kBlock, true>), dim3(a.num_nodes, (a.H + 3) / 4), dim3(256), 0, s, a);
}

template <int D, bool F16>
void launch_rows(TreeArgs a, int R, hipStream_t s) {
  if (R == 16) return launch_few<D, F16, 1>(a, s);
  if (R == 32) return launch_few<D, F16, 2>(a, s);
  a.workgroups = std::min(a.workgroups, wide_resident(D, F16));
  IRON_LAUNCH((tree4_wide_kernel<D, F16>), dim3(a.workgroups), dim3(256), 0, s, a);
  IRON_LAUNCH((tree_join_kernel<D, F16, 128, kWideBlock, true>), dim3(a.num_nodes, (a.H + 3) / 4), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace iron

using namespace iron;

extern "C" long long iron_tree_attention_int4_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int num_seqs,
                                                              int num_nodes, int max_nodes, int max_pages, int page_size) {
  return tree_workspace(resident, n_heads, n_kv_heads, head_dim, num_seqs, num_nodes, max_nodes, max_pages, page_size);
}

extern "C" int iron_tree_attention_int4(const void* q, const void* k_new, const void* v_new, const void* k_pages,
                                        const void* v_pages, const int* page_table, const int* seq_lens,
                                        const int* node_starts, const int* tree_mask, void* out, int dtype, int n_heads,
                                        int n_kv_heads, int head_dim, int num_pages, int page_size, int num_seqs,
                                        int max_pages, int num_nodes, int max_nodes, float scale, void* workspace,
                                        long long workspace_bytes, void* stream) {
  TreeArgs a;
  if (int rc = tree_call("iron_tree_attention_int4", resident, a, q, k_new, v_new, k_pages, v_pages, page_table, seq_lens,
                         node_starts, tree_mask, out, dtype, n_heads, n_kv_heads, head_dim, num_pages, page_size, num_seqs,
                         max_pages, num_nodes, max_nodes, scale, workspace, workspace_bytes))
    return rc;
  const int R = rows_of_tile(n_heads, n_kv_heads, max_nodes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64)
    dtype ? launch_rows<64, true>(a, R, s) : launch_rows<64, false>(a, R, s);
  else
    dtype ? launch_rows<128, true>(a, R, s) : launch_rows<128, false>(a, R, s);
  return check_launch("tree_attention_int4");
}
