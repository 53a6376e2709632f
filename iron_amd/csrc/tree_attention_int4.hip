// Attention of drafted trees over a paged KV cache of 4-bit rows (int4_rows.hpp):
// tree_attention.hip's mathematics, tiles and shares of work; the cached keys and
// values are b + s (16 + code), the tree's own are 16-bit rows.
#include "tree_common.hpp"

namespace iron {
namespace {

// One workgroup per node and 4 heads, a wave for each row, one key at a time.
template <int D, bool F16>
__global__ __launch_bounds__(256) void tree4_rows_kernel(TreeArgs a) {
  const int n = blockIdx.x, h = blockIdx.y * 4 + uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (h >= a.H) return;
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    const int s = min(s0 + lane, a.num_seqs - 1);
    int first, nodes;
    tree_of(a, s, first, nodes);
    const unsigned long long has = __ballot(s0 + lane < a.num_seqs && first <= n && n < first + nodes);
    if (!has) continue;
    const int who = s0 + __ffsll(has) - 1;
    attend_row<D, F16, true>(a, uniform_tiles_of<16, kBlock>(a, who), who, n, h);
    return;
  }
}

int resident(int D, int R) { return 512; }

template <int D, bool F16>
void launch_rows(const TreeArgs& a, hipStream_t s) {
  IRON_LAUNCH((tree4_rows_kernel<D, F16>), dim3(a.num_nodes, (a.H + 3) / 4), dim3(256), 0, s, a);
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64)
    dtype ? launch_rows<64, true>(a, s) : launch_rows<64, false>(a, s);
  else
    dtype ? launch_rows<128, true>(a, s) : launch_rows<128, false>(a, s);
  return check_launch("tree_attention_int4");
}
