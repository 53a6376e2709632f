// Which drafted tokens the target accepts.
//
// p(n) = softmax(logits[n] / T), q(n) = softmax(draft[n] / T). At an accepted
// node, with w_0 = p and R_0 = 1, its child j (in row order, token x, number u) is
// accepted if u q(x) < w_j(x) / R_j; else w_{j+1} = max(w_j / R_j - q, 0) and
// R_{j+1} is its sum. Where none is, the next token is drawn from w: the first x
// whose cumulative sum passes r sum(w). Unrolled, w_j = max(a_j p - b_j q, 0) with
// a_{j+1} = a_j / R_j and b_{j+1} = b_j / R_j + 1, so that a node's state is two
// numbers and a sum over the vocabulary. Without draft logits q is 1 at the child's
// token: w is p without the tokens tried, and no sums are needed on the way.
//
// Everything is in 64 bits: a vocabulary of 2^17 tokens of like probability puts
// the borders of the cumulative sum 2^-17 apart, where sums of fp32 exponentials
// (off by 2^-24 each) would draw another token in some percent of the calls.
#include "iron_common.hpp"
#include "../../include/iron_hip.h"

#include <algorithm>
#include <cfloat>

namespace iron {
namespace {

constexpr int kChunk = 4096;  // logits of a workgroup
constexpr int kMaxNodes = 1024;
constexpr int kMaxSeqs = 8192;

struct RowStat {  // of a row, or of a chunk of it
  double z;       // sum of exp((l - m) / T)
  float m;        // the largest logit
  int best;       // its first index
};

struct Choice {  // what a sequence came to
  double a, b;   // weights max(a p - b q, 0)
  int node;      // the row whose distribution the next token is drawn from, -1 for an empty tree
  int count;     // accepted rows
  int tried;     // children that were not accepted there
  int pad;
};

struct VerifyArgs {
  const void* logits;  // (num_nodes, vocab)
  const void* draft;   // the same, or null
  const int* tokens;   // (num_nodes)
  const int* parents;  // (num_nodes), within the tree
  const int* starts;   // (num_seqs + 1)
  const float* temps;  // (num_seqs)
  const float* accept; // (num_nodes)
  const float* sample; // (num_seqs)
  int* rows;           // (num_nodes)
  int* row_starts;     // (num_seqs + 1)
  int* next;           // (num_seqs)
  RowStat* part;       // workspace (num_nodes [x 2], chunks)
  RowStat* stat;       // workspace (num_nodes [x 2])
  double* chance;      // workspace (num_nodes, 2): p and q of the parent's row at the node's token
  double2* ab;         // workspace (max_children, num_nodes): a_j, b_j
  double* mass;        // workspace (max_children, num_nodes, chunks): parts of R_j
  Choice* choice;      // workspace (num_seqs)
  double* weight;      // workspace (num_seqs, chunks): parts of the last sum(w)
  int* path;           // workspace (num_nodes): accepted rows, from each tree's first row on
  int vocab, num_seqs, num_nodes, max_nodes, max_children, chunks;
};

// The tree of sequence s: its first row and its nodes, cut to the arrays.
__device__ __forceinline__ void tree_of(const VerifyArgs& a, int s, int& first, int& nodes) {
  first = min(max(a.starts[s], 0), a.num_nodes);
  nodes = min(min(max(a.starts[s + 1], first), a.num_nodes) - first, a.max_nodes);
}

struct Place {
  int seq, first, nodes;
};

// The first sequence whose tree holds row n (seq -1: none). Every thread calls it.
__device__ __forceinline__ Place place_of(const VerifyArgs& a, int n, int* shared) {
  if (threadIdx.x == 0) *shared = a.num_seqs;
  __syncthreads();
  for (int s = threadIdx.x; s < a.num_seqs; s += blockDim.x) {
    int first, nodes;
    tree_of(a, s, first, nodes);
    if (first <= n && n < first + nodes) atomicMin(shared, s);
  }
  __syncthreads();
  Place p = {*shared, 0, 0};
  if (p.seq == a.num_seqs)
    p.seq = -1;
  else
    tree_of(a, p.seq, p.first, p.nodes);
  return p;
}

// Children of node i of a tree (whole workgroup). A parent comes before its child.
__device__ __forceinline__ int children_of(const VerifyArgs& a, const Place& p, int i, int* shared) {
  __syncthreads();
  if (threadIdx.x == 0) *shared = 0;
  __syncthreads();
  int mine = 0;
  for (int c = i + 1 + threadIdx.x; c < p.nodes; c += blockDim.x) mine += a.parents[p.first + c] == i;
  if (mine) atomicAdd(shared, mine);
  __syncthreads();
  return *shared;
}

// A temperature that is not above 0 stands for the likeliest token.
__device__ __forceinline__ bool greedy(float t) { return !(t > 0.f); }

// A logit as it counts: NaN is none, an infinity the largest number.
__device__ __forceinline__ float logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

template <typename T>
__device__ __forceinline__ float load(const void* base, long long i) {
  const T x = static_cast<const T*>(base)[i];
  if constexpr (std::is_same_v<T, uint16_t>) return logit(bf16_to_f32(x));
  else return logit(static_cast<float>(x));
}

__device__ __forceinline__ double boost(float l, float m, double inv_t) { return l == -INFINITY ? 0. : exp((static_cast<double>(l) - m) * inv_t); }

__device__ __forceinline__ double wave_sum64(double x) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}

// Sum over the workgroup's 256 threads, in the same order every time. Every thread calls it.
__device__ __forceinline__ double block_sum(double x, double* tmp) {
  x = wave_sum64(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = x;
  __syncthreads();
  return (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
}

// One chunk of a row of target or draft logits: its maximum and its sum.
template <typename T>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ int si;
  __shared__ double tmp[4];
  __shared__ float top[4];
  __shared__ int arg[4];
  const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks;
  const bool target = row < a.num_nodes;
  const int n = target ? row : row - a.num_nodes;
  const Place p = place_of(a, n, &si);
  if (p.seq < 0) return;
  const float temp = a.temps[p.seq];
  if (!target && (greedy(temp) || children_of(a, p, n - p.first, &si) == 0)) return;
  const void* base = target ? a.logits : a.draft;
  const long long at = static_cast<long long>(n) * a.vocab;
  const int lo = c * kChunk, hi = min(lo + kChunk, a.vocab);
  float l[kChunk / 256];
  float m = -INFINITY;
  int best = INT_MAX;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    const int x = lo + i * 256 + static_cast<int>(threadIdx.x);
    l[i] = x < hi ? load<T>(base, at + x) : -INFINITY;
    if (l[i] > m) {
      m = l[i];
      best = x;
    }
  }
  const float wm = wave_max(m);
  int wb = m == wm ? best : INT_MAX;
  for (int d = 32; d; d >>= 1) wb = min(wb, __shfl_xor(wb, d, 64));
  if ((threadIdx.x & 63) == 0) {
    top[threadIdx.x >> 6] = wm;
    arg[threadIdx.x >> 6] = wb;
  }
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  best = INT_MAX;
  for (int w = 0; w < 4; ++w)
    if (top[w] == m) best = min(best, arg[w]);
  double z = 0.;
  if (!greedy(temp)) {
    const double inv = 1. / temp;
#pragma unroll
    for (int i = 0; i < kChunk / 256; ++i) z += boost(l[i], m, inv);
    z = block_sum(z, tmp);
  }
  if (threadIdx.x == 0) a.part[static_cast<long long>(row) * a.chunks + c] = {z, m, best};
}

// The chunks of a row together (one wave).
__device__ __forceinline__ RowStat merge(const VerifyArgs& a, int row, double inv) {
  const int lane = threadIdx.x & 63;
  const RowStat* part = a.part + static_cast<long long>(row) * a.chunks;
  float m = -INFINITY;
  for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, part[c].m);
  m = wave_max(m);
  double z = 0.;
  int best = INT_MAX;
  for (int c = lane; c < a.chunks; c += 64) {
    const RowStat r = part[c];
    z += r.z * boost(r.m, m, inv);
    if (r.m == m) best = min(best, r.best);
  }
  for (int d = 32; d; d >>= 1) best = min(best, __shfl_xor(best, d, 64));
  return {wave_sum64(z), m, m == -INFINITY ? -1 : best};
}

// One wave per node: its rows' sums, and the probabilities of its token in its parent's.
template <typename T>
__global__ __launch_bounds__(64) void verify_merge_kernel(VerifyArgs a) {
  __shared__ int si;
  const int n = blockIdx.x, lane = threadIdx.x;
  const Place p = place_of(a, n, &si);
  if (p.seq < 0) return;
  const float temp = a.temps[p.seq];
  const double inv = greedy(temp) ? 0. : 1. / temp;
  const RowStat mine = merge(a, n, inv);
  if (lane == 0) a.stat[n] = mine;
  if (greedy(temp)) return;
  if (a.draft && children_of(a, p, n - p.first, &si)) {
    const RowStat q = merge(a, a.num_nodes + n, inv);
    if (lane == 0) a.stat[a.num_nodes + n] = q;
  }
  const int up = a.parents[n], x = a.tokens[n];
  if (n == p.first || up < 0 || up >= n - p.first) return;
  const int parent = p.first + up;
  const bool real = static_cast<unsigned>(x) < static_cast<unsigned>(a.vocab);
  const RowStat sp = merge(a, parent, inv);
  double pc = real && sp.z > 0. ? boost(load<T>(a.logits, static_cast<long long>(parent) * a.vocab + x), sp.m, inv) / sp.z : 0., qc = 1.;
  if (a.draft) {
    const RowStat sq = merge(a, a.num_nodes + parent, inv);
    qc = real && sq.z > 0. ? boost(load<T>(a.draft, static_cast<long long>(parent) * a.vocab + x), sq.m, inv) / sq.z : 0.;
  }
  if (lane == 0) {
    a.chance[2 * n] = pc;
    a.chance[2 * n + 1] = qc;
  }
}

// R_j of a row from its parts (one wave, every lane returns it).
__device__ __forceinline__ double mass_of(const VerifyArgs& a, int j, int n) {
  if (j == 0) return 1.;
  double r = 0.;
  const double* part = a.mass + (static_cast<long long>(j) * a.num_nodes + n) * a.chunks;
  for (int c = threadIdx.x & 63; c < a.chunks; c += 64) r += part[c];
  return wave_sum64(r);
}

// The weight of logit x of row n for a_j, b_j.
struct Weigh {
  double ka, kb, inv;  // a / sum, b / sum of p's and q's exponentials
  float mp, mq;
  __device__ __forceinline__ double operator()(float lp, float lq) const {
#pragma clang fp contract(off)  // equal rows of target and draft leave nothing at all
    return fmax(ka * boost(lp, mp, inv) - kb * boost(lq, mq, inv), 0.);
  }
};
__device__ __forceinline__ Weigh weigh(const VerifyArgs& a, int n, double ca, double cb, float temp) {
  const RowStat p = a.stat[n];
  Weigh w = {p.z > 0. ? ca / p.z : 0., 0., 1. / temp, p.m, 0.f};
  if (cb != 0.) {
    const RowStat q = a.stat[a.num_nodes + n];
    w.kb = q.z > 0. ? cb / q.z : 0.;
    w.mq = q.m;
  }
  return w;
}

// R_j's part of a chunk, for rows with more than j children.
template <typename T>
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs a, int j) {
  __shared__ int si;
  __shared__ double tmp[4];
  const int n = blockIdx.x / a.chunks, c = blockIdx.x - n * a.chunks;
  const Place p = place_of(a, n, &si);
  if (p.seq < 0) return;
  const float temp = a.temps[p.seq];
  if (greedy(temp) || children_of(a, p, n - p.first, &si) <= j) return;
  const double r = mass_of(a, j - 1, n);
  const double2 was = j == 1 ? make_double2(1., 0.) : a.ab[static_cast<long long>(j - 1) * a.num_nodes + n];
  const double2 now = make_double2(was.x / r, was.y / r + 1.);
  if (c == 0 && threadIdx.x == 0) a.ab[static_cast<long long>(j) * a.num_nodes + n] = now;
  const Weigh w = weigh(a, n, now.x, now.y, temp);
  const long long at = static_cast<long long>(n) * a.vocab;
  const int lo = c * kChunk, hi = min(lo + kChunk, a.vocab);
  double sum = 0.;
  for (int x = lo + static_cast<int>(threadIdx.x); x < hi; x += 256) sum += w(load<T>(a.logits, at + x), load<T>(a.draft, at + x));
  sum = block_sum(sum, tmp);
  if (threadIdx.x == 0) a.mass[(static_cast<long long>(j) * a.num_nodes + n) * a.chunks + c] = sum;
}

// Down a tree: which rows are accepted, and what the next token is drawn from
// (one wave, the same result in every workgroup that asks). path may be null.
__device__ Choice walk(const VerifyArgs& a, const Place& p, float temp, int* path) {
  const int lane = threadIdx.x & 63;
  Choice r = {1., 0., -1, 0, 0, 0};
  if (p.nodes == 0) return r;
  auto reach = [&](int i) {
    if (path && lane == 0) path[r.count] = p.first + i;
    r.count += 1;
    r.node = p.first + i;
    r.a = 1.;
    r.b = 0.;
    r.tried = 0;
  };
  reach(0);
  double left = 1.;  // R of the next child's test
  for (int i0 = 1; i0 < p.nodes; i0 += 64) {
    const int i = i0 + lane;
    const int up = i < p.nodes ? a.parents[p.first + i] : -1;
    int from = i0;
    while (true) {  // the next child of the current node
      const unsigned long long kids = __ballot(up == r.node - p.first && i >= from && i < p.nodes);
      if (!kids) break;
      const int k = i0 + __ffsll(kids) - 1, n = p.first + k;
      from = k + 1;
      if (r.tried >= a.max_children) continue;
      bool yes;
      if (greedy(temp)) {
        const int best = a.stat[r.node].best;
        yes = best >= 0 && best == a.tokens[n];
      } else {
        const double pc = a.chance[2 * n], qc = a.chance[2 * n + 1];
        if (a.draft) {
          yes = static_cast<double>(a.accept[n]) * qc < fmax(r.a * pc - r.b * qc, 0.) / left;
        } else {  // its token may have been tried before
          bool again = false;
          for (int e = lane; e < k; e += 64) again |= a.parents[p.first + e] == r.node - p.first && e > r.node - p.first && a.tokens[p.first + e] == a.tokens[n];
          again = __ballot(again) != 0;
          yes = !again && static_cast<double>(a.accept[n]) < pc / left;
          if (!yes && !again) left -= pc;
        }
      }
      if (yes) {
        reach(k);
        left = 1.;
      } else {
        r.tried += 1;
        if (a.draft && !greedy(temp)) {
          r.a /= left;
          r.b = r.b / left + 1.;
          left = r.tried < a.max_children ? mass_of(a, r.tried, r.node) : 1.;
          if (left == 0.) r.tried = a.max_children;  // nothing is left to accept
        }
      }
    }
  }
  return r;
}

// The weight of a token without draft logits: 0 for those that were tried.
__device__ __forceinline__ bool tried(const VerifyArgs& a, const Place& p, const Choice& r, int x) {
  if (a.draft) return false;
  int left = r.tried;
  for (int k = r.node - p.first + 1; k < p.nodes && left; ++k)
    if (a.parents[p.first + k] == r.node - p.first) {
      if (a.tokens[p.first + k] == x) return true;
      --left;
    }
  return false;
}

// Sequence s's walk, and a chunk of the sum that its next token is drawn by.
template <typename T>
__global__ __launch_bounds__(256) void verify_walk_kernel(VerifyArgs a) {
  __shared__ Choice sr;
  __shared__ double tmp[4];
  const int s = blockIdx.x / a.chunks, c = blockIdx.x - s * a.chunks;
  Place p = {s, 0, 0};
  tree_of(a, s, p.first, p.nodes);
  const float temp = a.temps[s];
  if (threadIdx.x < 64) {
    const Choice r = walk(a, p, temp, c == 0 ? a.path + p.first : nullptr);
    if (threadIdx.x == 0) {
      sr = r;
      if (c == 0) a.choice[s] = r;
    }
  }
  __syncthreads();
  const Choice r = sr;
  if (r.node < 0 || greedy(temp)) return;
  const Weigh w = weigh(a, r.node, r.a, r.b, temp);
  const long long at = static_cast<long long>(r.node) * a.vocab;
  const int lo = c * kChunk, hi = min(lo + kChunk, a.vocab);
  double sum = 0.;
  for (int x = lo + static_cast<int>(threadIdx.x); x < hi; x += 256)
    if (!tried(a, p, r, x)) sum += w(load<T>(a.logits, at + x), r.b != 0. ? load<T>(a.draft, at + x) : -INFINITY);
  sum = block_sum(sum, tmp);
  if (threadIdx.x == 0) a.weight[static_cast<long long>(s) * a.chunks + c] = sum;
}

// One workgroup per sequence: its rows' place in the result, and its next token.
template <typename T>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a) {
  __shared__ int before, total, found, last;
  __shared__ int at_chunk;
  __shared__ double goal, base;
  __shared__ double scan[256], tmp[4];
  static_assert((1 << 20) / kChunk <= 256, "a thread to each chunk of the largest vocabulary");
  const int s = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) before = total = 0;
  __syncthreads();
  int b = 0, t = 0;
  for (int i = tid; i < a.num_seqs; i += 256) {
    const int n = a.choice[i].count;
    t += n;
    if (i < s) b += n;
  }
  if (t) atomicAdd(&total, t);
  if (b) atomicAdd(&before, b);
  __syncthreads();
  Choice r = a.choice[s];
  Place p = {s, 0, 0};
  tree_of(a, s, p.first, p.nodes);
  for (int i = tid; i < r.count && before + i < a.num_nodes; i += 256) a.rows[before + i] = a.path[p.first + i];
  for (long long i = total + s * 256LL + tid; i < a.num_nodes; i += a.num_seqs * 256LL) a.rows[i] = -1;
  if (tid == 0) {
    a.row_starts[s] = before;
    if (s == a.num_seqs - 1) a.row_starts[a.num_seqs] = total;
  }
  const float temp = a.temps[s];
  if (r.node < 0 || greedy(temp)) {
    if (tid == 0) a.next[s] = r.node < 0 ? -1 : a.stat[r.node].best;
    return;
  }
  const RowStat all = a.stat[r.node];
  const double inv = 1. / temp;
  // the chunks' weights; where nothing is left of p, p's own
  double x = tid < a.chunks ? a.weight[static_cast<long long>(s) * a.chunks + tid] : 0.;
  double sum = 0.;
  const bool rest = block_sum(x, tmp) > 0.;
  if (!rest) {
    r.a = 1., r.b = 0., r.tried = 0;
    if (tid < a.chunks) {
      const RowStat part = a.part[static_cast<long long>(r.node) * a.chunks + tid];
      x = all.z > 0. ? part.z * boost(part.m, all.m, inv) / all.z : 0.;
    }
  }
  scan[tid] = x;
  __syncthreads();
  if (tid == 0) {
    sum = 0.;
    for (int c = 0; c < a.chunks; ++c) sum += scan[c];
    goal = a.sample[s] * sum;
    double run = 0.;
    int k = -1;
    for (int c = 0; c < a.chunks; ++c) {
      if (scan[c] > 0.) {
        k = c;
        base = run;
        if (run + scan[c] > goal) break;
      }
      run += scan[c];
    }
    at_chunk = k;
    found = INT_MAX;
    last = -1;
  }
  __syncthreads();
  if (at_chunk < 0) {
    if (tid == 0) a.next[s] = -1;
    return;
  }
  const Weigh w = weigh(a, r.node, r.a, r.b, temp);
  const long long at = static_cast<long long>(r.node) * a.vocab;
  const int lo = at_chunk * kChunk + tid * (kChunk / 256), hi = min(lo + kChunk / 256, a.vocab);
  double mine[kChunk / 256];
  sum = 0.;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    const int x = lo + i;
    mine[i] = x < hi && !tried(a, p, r, x) ? w(load<T>(a.logits, at + x), r.b != 0. ? load<T>(a.draft, at + x) : -INFINITY) : 0.;
    sum += mine[i];
  }
  scan[tid] = sum;
  __syncthreads();
  for (int d = 1; d < 256; d *= 2) {
    const double y = tid >= d ? scan[tid - d] : 0.;
    __syncthreads();
    scan[tid] += y;
    __syncthreads();
  }
  double run = base + (tid ? scan[tid - 1] : 0.);
  int hit = INT_MAX, end = -1;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    run += mine[i];
    if (mine[i] > 0.) {
      end = lo + i;
      if (hit == INT_MAX && run > goal) hit = lo + i;
    }
  }
  if (hit != INT_MAX) atomicMin(&found, hit);
  if (end >= 0) atomicMax(&last, end);
  __syncthreads();
  if (tid == 0) a.next[s] = found != INT_MAX ? found : last;
}

const char* check_shape(int vocab, int num_seqs, int num_nodes, int max_nodes, int max_children) {
  if (vocab < 1 || vocab > (1 << 20)) return "vocab outside [1, 2^20]";
  if (num_seqs < 1 || num_seqs > kMaxSeqs) return "num_seqs outside [1, 8192]";
  if (num_nodes < 1 || num_nodes > (1 << 20)) return "num_nodes outside [1, 2^20]";
  if (max_nodes < 1 || max_nodes > kMaxNodes) return "max_nodes outside [1, 1024]";
  if (max_children < 1 || max_children > 64) return "max_children outside [1, 64]";
  const long long chunks = (vocab + kChunk - 1) / kChunk;
  if (num_nodes * chunks >= (1LL << 23)) return "num_nodes * vocab: chunks of 4096 logits must count below 2^23";  // a launch has less than 2^32 threads
  return nullptr;
}

// The workspace's parts, from `base` on; returns its bytes.
long long lay_out(VerifyArgs& a, bool draft, char* base) {
  long long at = 0;
  auto take = [&](auto*& p, long long n) {
    p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
    at += (n * sizeof(*p) + 15) / 16 * 16;
  };
  const long long rows = (draft ? 2LL : 1LL) * a.num_nodes;
  take(a.part, rows * a.chunks);
  take(a.stat, rows);
  take(a.chance, 2LL * a.num_nodes);
  take(a.choice, a.num_seqs);
  take(a.weight, static_cast<long long>(a.num_seqs) * a.chunks);
  take(a.path, a.num_nodes);
  const long long sums = draft && a.max_children > 1 ? static_cast<long long>(a.max_children) * a.num_nodes : 0;
  take(a.ab, sums);
  take(a.mass, sums * a.chunks);
  return at;
}

template <typename T>
void launch(const VerifyArgs& a, hipStream_t s) {
  const int rows = (a.draft ? 2 : 1) * a.num_nodes;
  IRON_LAUNCH((verify_stats_kernel<T>), dim3(rows * a.chunks), dim3(256), 0, s, a);
  IRON_LAUNCH((verify_merge_kernel<T>), dim3(a.num_nodes), dim3(64), 0, s, a);
  if (a.draft)
    for (int j = 1; j < a.max_children; ++j) IRON_LAUNCH((verify_mass_kernel<T>), dim3(a.num_nodes * a.chunks), dim3(256), 0, s, a, j);
  IRON_LAUNCH((verify_walk_kernel<T>), dim3(a.num_seqs * a.chunks), dim3(256), 0, s, a);
  IRON_LAUNCH((verify_draw_kernel<T>), dim3(a.num_seqs), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace iron

using namespace iron;

extern "C" long long iron_draft_verify_workspace_bytes(int vocab, int num_seqs, int num_nodes, int max_nodes, int max_children,
                                                       int draft) {
  if (check_shape(vocab, num_seqs, num_nodes, max_nodes, max_children)) return -1;
  VerifyArgs a = {};
  a.num_nodes = num_nodes;
  a.num_seqs = num_seqs;
  a.max_children = max_children;
  a.chunks = (vocab + kChunk - 1) / kChunk;
  return lay_out(a, draft != 0, nullptr);
}

extern "C" int iron_draft_verify(const void* logits, const void* draft_logits, const int* tokens, const int* parents,
                                 const int* node_starts, const float* temperatures, const float* accept_draws,
                                 const float* sample_draws, int* rows, int* row_starts, int* next_tokens, int dtype, int vocab,
                                 int num_seqs, int num_nodes, int max_nodes, int max_children, void* workspace,
                                 long long workspace_bytes, void* stream) {
  const char* who = "iron_draft_verify";
  const char* bad = check_shape(vocab, num_seqs, num_nodes, max_nodes, max_children);
  IRON_REQUIRE(!bad, "%s: %s", who, bad);
  IRON_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype=%d is none of 0 (bf16), 1 (fp16) and 2 (fp32)", who, dtype);
  IRON_REQUIRE(logits && aligned16(logits) && aligned16(draft_logits), "%s: logits must be given and 16-byte aligned", who);
  for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(parents), static_cast<const void*>(node_starts),
                        static_cast<const void*>(temperatures), static_cast<const void*>(accept_draws), static_cast<const void*>(sample_draws),
                        static_cast<const void*>(rows), static_cast<const void*>(row_starts), static_cast<const void*>(next_tokens)})
    IRON_REQUIRE(p && (reinterpret_cast<uintptr_t>(p) & 3u) == 0, "%s: arrays of 4-byte numbers must be given and 4-byte aligned", who);
  const long long need = iron_draft_verify_workspace_bytes(vocab, num_seqs, num_nodes, max_nodes, max_children, draft_logits != nullptr);
  IRON_REQUIRE(workspace && aligned16(workspace), "%s: the workspace must be given and 16-byte aligned", who);
  IRON_REQUIRE(workspace_bytes >= need, "%s: workspace of %lld bytes, %lld needed", who, workspace_bytes, need);
  VerifyArgs a = {};
  a.logits = logits;
  a.draft = draft_logits;
  a.tokens = tokens;
  a.parents = parents;
  a.starts = node_starts;
  a.temps = temperatures;
  a.accept = accept_draws;
  a.sample = sample_draws;
  a.rows = rows;
  a.row_starts = row_starts;
  a.next = next_tokens;
  a.vocab = vocab;
  a.num_seqs = num_seqs;
  a.num_nodes = num_nodes;
  a.max_nodes = max_nodes;
  a.max_children = max_children;
  a.chunks = (vocab + kChunk - 1) / kChunk;
  lay_out(a, draft_logits != nullptr, static_cast<char*>(workspace));
  hipStream_t s = static_cast<hipStream_t>(stream);
  dtype == 0 ? launch<uint16_t>(a, s) : dtype == 1 ? launch<_Float16>(a, s) : launch<float>(a, s);
  return check_launch("draft_verify");
}
