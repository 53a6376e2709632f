// Attention of drafted trees over a paged KV cache.
//
// out[i,h] = sum_j softmax_j(scale q[i,h] . k_j) v_j over the cached positions
// of node i's sequence and the nodes of its tree that it sees.
#include "iron_common.hpp"
#include "../../include/iron_hip.h"

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
  int H, Hkv, num_pages, page_shift, num_seqs, max_pages, num_nodes, max_nodes, words;
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

// One workgroup of 4 waves per (node of a tree, head): each wave takes every
// fourth key, a lane D / 64 dims.
template <int D, bool F16>
__global__ __launch_bounds__(256) void tree_attention_kernel(TreeArgs a) {
  __shared__ float part[4][D + 2];
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int s = blockIdx.z, h = blockIdx.y, hk = h / (a.H / a.Hkv);
  int first, nodes;
  tree_of(a, s, first, nodes);
  if (static_cast<int>(blockIdx.x) >= nodes) return;
  const long long row = first + blockIdx.x;
  const int ps = 1 << a.page_shift;
  const int len = min(max(a.lens[s], 0), a.max_pages * ps);
  float q[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    q[e] = widen<F16>(a.q[(row * a.H + h) * D + lane * E + e]);
    o[e] = 0.f;
  }
  for (int j = w; j < len + nodes; j += 4) {
    const uint16_t *k, *v;
    if (j < len) {
      const int page = a.table[static_cast<long long>(s) * a.max_pages + (j >> a.page_shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_pages)) continue;
      const long long at = ((static_cast<long long>(page) * a.Hkv + hk) * ps + (j & (ps - 1))) * D;
      k = a.k_pages + at;
      v = a.v_pages + at;
    } else {
      const int n = j - len;
      if (!(a.mask[row * a.words + (n >> 5)] >> (n & 31) & 1)) continue;
      const long long at = (static_cast<long long>(first + n) * a.Hkv + hk) * D;
      k = a.k_new + at;
      v = a.v_new + at;
    }
    float x = 0.f;
    for (int e = 0; e < E; ++e) x += q[e] * widen<F16>(k[lane * E + e]);
    x = wave_sum(x) * a.scale_log2;
    const float top = fmaxf(m, x);
    const float off = top == -INFINITY ? 0.f : top;
    const float alpha = exp2f(m - off), p = exp2f(x - off);
    m = top;
    l = l * alpha + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + p * widen<F16>(v[lane * E + e]);
  }
  for (int e = 0; e < E; ++e) part[w][lane * E + e] = o[e];
  if (lane == 0) {
    part[w][D] = m;
    part[w][D + 1] = l;
  }
  __syncthreads();
  if (w) return;
  float top = -INFINITY, sum = 0.f, r[E] = {};
  for (int i = 0; i < 4; ++i) top = fmaxf(top, part[i][D]);
  for (int i = 0; i < 4; ++i) {
    const float f = top == -INFINITY ? 0.f : exp2f(part[i][D] - top);
    sum += f * part[i][D + 1];
    for (int e = 0; e < E; ++e) r[e] += f * part[i][lane * E + e];
  }
  for (int e = 0; e < E; ++e) a.out[(row * a.H + h) * D + lane * E + e] = narrow<F16>(sum > 0.f || sum != sum ? r[e] / sum : 0.f);
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
  return nullptr;
}

}  // namespace
}  // namespace iron

using namespace iron;

extern "C" long long iron_tree_attention_workspace_bytes(int n_heads, int n_kv_heads, int head_dim, int num_seqs,
                                                         int num_nodes, int max_nodes, int max_pages, int page_size) {
  if (check_shape(n_heads, n_kv_heads, head_dim, num_seqs, num_nodes, max_nodes, max_pages, page_size)) return -1;
  return 16;
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
  IRON_REQUIRE(out != q && out != k_new && out != v_new, "%s: out is one of the inputs", who);
  IRON_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale=%g must be positive and finite", who, scale);
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
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctz(page_size);
  a.num_seqs = num_seqs;
  a.max_pages = max_pages;
  a.num_nodes = num_nodes;
  a.max_nodes = max_nodes;
  a.words = (max_nodes + 31) / 32;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(max_nodes, n_heads, num_seqs), block(256);
  if (head_dim == 64) {
    if (dtype)
      IRON_LAUNCH((tree_attention_kernel<64, true>), grid, block, 0, s, a);
    else
      IRON_LAUNCH((tree_attention_kernel<64, false>), grid, block, 0, s, a);
  } else {
    if (dtype)
      IRON_LAUNCH((tree_attention_kernel<128, true>), grid, block, 0, s, a);
    else
      IRON_LAUNCH((tree_attention_kernel<128, false>), grid, block, 0, s, a);
  }
  return check_launch("tree_attention");
}
