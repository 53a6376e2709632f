// Which drafted tokens the target accepts.
//
// p(n) = softmax(logits[n] / T), q(n) = softmax(draft[n] / T). At an accepted
// node, with w_0 = p and R_0 = 1, its child j (in row order, token x, number u) is
// accepted if u q(x) < w_j(x) / R_j; else w_{j+1} = max(w_j / R_j - q, 0) and
// R_{j+1} is its sum. Where none is, the next token is drawn from w: the first x
// whose cumulative sum passes r sum(w). A node's state is the numbers 1 / R_i; every
// token's w is taken through them step by step, two instructions each. (Unrolled it is
// max(a p - b q, 0) with two numbers, but where little is left, a and b are large and
// all of it cancels: rows with nearly all of their probability at one token came out wrong.)
// Without draft logits q is 1 at the child's token: w is p without the tokens tried,
// and no sums are needed on the way unless these have nearly all of p.
//
// Everything is in 64 bits: a vocabulary of 2^17 tokens of like probability puts
// the borders of the cumulative sum 2^-17 apart, where sums of fp32 exponentials
// (off by 2^-24 each) draw another token in 0.3 % of the calls (0.2 % for 128256
// tokens of ordinary rows; 12,000 draws each).
#include "iron_common.hpp"
#include "../../include/iron_hip.h"

#include <algorithm>
#include <cfloat>

namespace iron {
namespace {

constexpr int kSub = 1024;  // logits of a wave (with two such parts to a wave, one behind the other, whole calls took 1 % less to 3 % more)
constexpr int kWalk = 4 * kSub;  // of a workgroup that sums the last weights
constexpr int kMaxNodes = 1024;
constexpr int kMaxSeqs = 8192;

struct RowStat {  // of a row, or of a part of it
  double z;       // sum of exp((l - m) / T)
  float m;        // the largest logit
  int best;       // its first index, -1 where no logit counts
};

struct Choice {  // what a sequence came to
  int node;   // the row whose distribution the next token is drawn from, -1 for an empty tree
  int count;  // accepted rows
  int tried;  // children that were not accepted there
  int steps;  // with draft logits: how many of them were taken off p
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
  RowStat* part;       // workspace (num_nodes [x 2], subs)
  RowStat* stat;       // workspace (num_nodes [x 2])
  double2* chance;     // workspace (num_nodes): p and q of the parent's row at the node's token
  double* scale;       // workspace (max_children - 1, num_nodes): 1 / R_j from j = 0 on; below 0 where a child up to the j-th is accepted
  double* mass;        // workspace (max_children - 1, num_nodes, subs): parts of R_j from j = 1 on
  Choice* choice;      // workspace (num_seqs)
  double* weight;      // workspace (num_seqs, subs): parts of the last sum(w)
  int* path;           // workspace (num_nodes): accepted rows, from each tree's first row on
  int* tried;          // workspace (num_seqs, max_children): tokens that were not accepted at the last node
  double* last;        // workspace (num_seqs, max_children): 1 / R_j there
  int vocab, num_seqs, num_nodes, max_nodes, max_children;
  int subs;            // parts of kSub places in a row, made up to whole fours
};

// The same value in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A tree: its sequence (-1: none), its first row and its nodes, cut to the arrays.
struct Tree {
  int seq, first, nodes;
};

__device__ __forceinline__ Tree tree_of(const VerifyArgs& a, int s) {
  const int first = min(max(a.starts[s], 0), a.num_nodes);
  return {s, uniform(first), uniform(min(min(max(a.starts[s + 1], first), a.num_nodes) - first, a.max_nodes))};
}

// The tree of row n, the last one that begins at or before it: 64 entries of starts
// at a time, by every wave for itself.
__device__ __forceinline__ Tree tree_with(const VerifyArgs& a, int n) {
  const int lane = threadIdx.x & 63;
  int lo = 0, count = a.num_seqs;  // the sequence is one of lo .. lo + count - 1
  while (count > 1) {
    const int step = (count + 63) / 64, at = lane * step;
    const unsigned long long before = __ballot(at < count && a.starts[lo + min(at, count - 1)] <= n);
    const int k = max(__popcll(before) - 1, 0);
    lo += k * step;
    count = min(step, count - k * step);
  }
  Tree t = tree_of(a, lo);
  if (n < t.first || n >= t.first + t.nodes) t.seq = -1;
  return t;
}

// Children of node i of a tree (a wave). A parent comes before its child.
__device__ __forceinline__ int children_of(const VerifyArgs& a, const Tree& t, int i) {
  int n = 0;
  for (int c0 = i + 1; c0 < t.nodes; c0 += 64) {
    const int c = c0 + (threadIdx.x & 63);
    n += __popcll(__ballot(c < t.nodes && a.parents[t.first + min(c, t.nodes - 1)] == i));
  }
  return n;
}

// A temperature that is not above 0 stands for the likeliest token.
__device__ __forceinline__ bool greedy(float t) { return !(t > 0.f); }

// A logit as it counts: NaN is none, an infinity the largest number.
__device__ __forceinline__ float logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

template <typename T>
__device__ __forceinline__ float widen(T x) {
  if constexpr (std::is_same_v<T, uint16_t>) return bf16_to_f32(x);
  else return static_cast<float>(x);
}

// Rows need no alignment but their elements': a row's places are counted from the
// 16-byte boundary at or before it, so that the lanes of all rows load 16 bytes each;
// place x holds token x - shift. What is fetched is made numbers only where it is
// used, so that fetches stay in flight until then.
template <typename T>
struct Row {
  const T* base;
  int shift, end;  // places [shift, end) are the row's
  int limit;       // up to here a whole vector of 16 bytes is the buffer's
  template <int N>
  struct alignas(N * sizeof(T)) Vec {
    T e[N];
  };
  __device__ __forceinline__ Row(const VerifyArgs& a, const void* logits, int n) {
    const T* row = static_cast<const T*>(logits) + static_cast<long long>(n) * a.vocab;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
    base = row - shift;
    end = shift + a.vocab;
    const long long left = static_cast<long long>(a.num_nodes - n) * a.vocab + shift;
    limit = static_cast<int>(min(left, 1LL << 30)) - 16 / static_cast<int>(sizeof(T));
  }
  // N places from x on, a multiple of N; anything where they are not the row's
  template <int N>
  __device__ __forceinline__ Vec<N> fetch(int x) const {
    if (limit < 0) return {};  // a buffer of less than 16 bytes
    return *reinterpret_cast<const Vec<N>*>(base + min(x, limit / N * N));
  }
  // Their logits as they are, -inf outside the row; `inside`: all of them are the row's and the buffer has them whole
  template <int N>
  __device__ __forceinline__ void expand(int x, const Vec<N>& v, bool inside, float (&l)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = widen(v.e[i]);
    if (!inside) {
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = x + i >= shift && x + i < end ? l[i] : -INFINITY;
      if (x > limit && x < end)  // the last ones of the buffer
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (x + i >= shift && x + i < end) l[i] = widen(base[x + i]);
    }
  }
  // Whether places [x, x + n) are all the row's and the buffer has their vectors whole.
  __device__ __forceinline__ bool inside(int x, int n) const { return x >= shift && x + n <= min(end, limit); }
  __device__ __forceinline__ float token(int x) const { return logit(widen(base[shift + x])); }
};

// The places of a lane in part `sub` of a row: kVecs loads of kVec.
template <typename T>
constexpr int kVec = 16 / sizeof(T);
template <typename T>
constexpr int kVecs = kSub / 64 / kVec<T>;
template <typename T>
__device__ __forceinline__ int place(int sub, int i) {
  return sub * kSub + (i * 64 + static_cast<int>(threadIdx.x & 63)) * kVec<T>;
}

// x moved across lanes by DPP control CTRL, 0 into lanes outside ROWMASK or without a source.
template <int CTRL, int ROWMASK = 0xf>
__device__ __forceinline__ double dpp64(double x) {
  const long long b = __builtin_bit_cast(long long, x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWMASK, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWMASK, 0xf, false);
  return __builtin_bit_cast(double, static_cast<long long>(hi) << 32 | lo);
}

__device__ __forceinline__ double lane64(double x, int lane) {
  const long long b = __builtin_bit_cast(long long, x);
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
  return __builtin_bit_cast(double, static_cast<long long>(hi) << 32 | lo);
}

// Inclusive sums over the wave's lanes, in the same order every time. All lanes are active.
__device__ __forceinline__ double wave_scan64(double x) {
  x += dpp64<0x111>(x);  // row_shr 1, 2, 4, 8, then the last lanes of rows into the rows behind
  x += dpp64<0x112>(x);
  x += dpp64<0x114>(x);
  x += dpp64<0x118>(x);
  x += dpp64<0x142, 0xa>(x);
  x += dpp64<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double wave_sum64(double x) { return lane64(wave_scan64(x), 63); }

// log2(e) / T.
__device__ __forceinline__ double rate_of(float temp) { return 1.4426950408889634 / temp; }

// exp((l - m) / T) for l <= m, 0 for l = -inf: 2^t as 2^n 2^f with f in [-1/2, 1/2], the
// series of 2^f to its 11th term (off by 2^-46.7 at most): 19 instructions of 5 cycles
// each, where the library's exp takes some 40. The terms stand in scalar registers:
// left to the compiler, each was moved into two vector registers before its use.
struct Exp2 {
  double k[12] = {1., 0x1.62e42fefa39efp-1, 0x1.ebfbdff82c58ep-3, 0x1.c6b08d704a0bfp-5, 0x1.3b2ab6fba4e77p-7, 0x1.5d87fe78a6730p-10, 0x1.430912f86c786p-13, 0x1.ffcbfc588b0c5p-17, 0x1.62c0223a5c822p-20, 0x1.b5253d395e7c1p-24, 0x1.e4cf5158b8ec7p-28, 0x1.e8cac7351bb22p-32};
  __device__ __forceinline__ Exp2() {
#pragma unroll
    for (int i = 0; i < 12; ++i) asm("" : "+s"(k[i]));
  }
  __device__ __forceinline__ double operator()(float l, float m, double rate) const {
    double t = (static_cast<double>(l) - m) * rate;
    t = __builtin_fmax(t, -1100.);  // 2^-1100 is 0
    const double n = rint(t), f = t - n;
    double y = fma(k[11], f, k[10]);
#pragma unroll
    for (int i = 9; i >= 0; --i) y = fma(y, f, k[i]);
    return __builtin_amdgcn_ldexp(y, static_cast<int>(n));
  }
  // Of N logits side by side: each step waits for the one before it, so a lone wave needs others in between.
  template <int N>
  __device__ __forceinline__ void operator()(const float (&l)[N], float m, double rate, double (&y)[N]) const {
    double f[N];
    int n[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const double t = __builtin_fmax((static_cast<double>(l[e]) - m) * rate, -1100.), r = rint(t);
      f[e] = t - r;
      n[e] = static_cast<int>(r);
      y[e] = fma(k[11], f[e], k[10]);
    }
#pragma unroll
    for (int i = 9; i >= 0; --i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = fma(y[e], f[e], k[i]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = __builtin_amdgcn_ldexp(y[e], n[e]);
  }
};

// The largest of three numbers, none of them NaN; the compiler's own makes quiet NaN of its operands first, at an instruction each.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// One part of a row of target or draft logits, by a wave: its maximum and its sum.
// Bound by the fp64 instructions (30.7 M logits, 8 trees of 26 nodes: 36 us, 24 of
// them these alone).
template <typename T>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  const int lane = threadIdx.x & 63;
  const int rows = a.draft ? 2 * a.num_nodes : a.num_nodes, id = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int row = id / a.subs, sub = id - row * a.subs;
  if (row >= rows) return;
  const bool target = row < a.num_nodes;
  const int n = target ? row : row - a.num_nodes;
  const Row<T> r(a, target ? a.logits : a.draft, n);
  typename Row<T>::template Vec<kVec<T>> raw[kVecs<T>];
  auto load = [&] {
#pragma unroll
    for (int i = 0; i < kVecs<T>; ++i) raw[i] = r.template fetch<kVec<T>>(place<T>(sub, i));
  };
  if (target) load();  // while the tree is looked up; of draft rows, many are not needed
  const Tree t = tree_with(a, n);
  if (t.seq < 0) return;
  const float temp = a.temps[t.seq];
  const bool top = greedy(temp);
  if (!target) {
    if (top || children_of(a, t, n - t.first) == 0) return;
    load();
  }
  const double rate = top ? 0. : rate_of(temp);
  const Exp2 boost;
  float x[kVecs<T>][kVec<T>], m = -INFINITY;
  const bool inside = r.inside(sub * kSub, kSub);
#pragma unroll
  for (int i = 0; i < kVecs<T>; ++i) r.expand(place<T>(sub, i), raw[i], inside, x[i]);
  auto clean = [&] {  // NaN and infinities as they count
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVecs<T>; ++i)
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e) m = fmaxf(m, x[i][e] = logit(x[i][e]));
    m = wave_max(m);
  };
  double z = 0.;
  int best = INT_MAX;
  if (top) {
    clean();
#pragma unroll
    for (int i = kVecs<T> - 1; i >= 0; --i)
#pragma unroll
      for (int e = kVec<T> - 1; e >= 0; --e) best = x[i][e] == m ? place<T>(sub, i) + e - r.shift : best;
    for (int d = 32; d; d >>= 1) best = min(best, __shfl_xor(best, d, 64));
  } else {
    // A signalling NaN would make v_max3 forget what came before it, so NaN are looked for on their own.
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kVecs<T>; ++i)
#pragma unroll
      for (int e = 0; e < kVec<T>; e += 2) {
        nan |= __builtin_isunordered(x[i][e], x[i][e + 1]);
        m = max3(m, x[i][e], x[i][e + 1]);
      }
    m = wave_max(m);
    if (__ballot(nan) || m == INFINITY) clean();
    if (m != -INFINITY)
#pragma unroll
      for (int i = 0; i < kVecs<T>; ++i) {
        double y[kVec<T>];
        boost(x[i], m, rate, y);
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e) z += y[e];
      }
    z = wave_sum64(z);
  }
  if (lane == 0) a.part[static_cast<long long>(row) * a.subs + sub] = {z, m, best};
}

// The parts of a row together (one wave). The first 256 stay in registers.
__device__ __forceinline__ RowStat merge(const VerifyArgs& a, int row, double rate) {
  constexpr int kHeld = 4;
  const int lane = threadIdx.x & 63;
  const Exp2 boost;
  const RowStat* part = a.part + static_cast<long long>(row) * a.subs;
  RowStat held[kHeld];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held[i] = i * 64 + lane < a.subs ? part[i * 64 + lane] : RowStat{0., -INFINITY, INT_MAX};
    m = fmaxf(m, held[i].m);
  }
  for (int c = kHeld * 64 + lane; c < a.subs; c += 64) m = fmaxf(m, part[c].m);
  m = wave_max(m);
  double z = 0.;
  int best = INT_MAX;
  auto add = [&](const RowStat& r) {
    z += r.z > 0. ? r.z * boost(r.m, m, rate) : 0.;
    if (r.m == m) best = min(best, r.best);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) add(held[i]);
  for (int c = kHeld * 64 + lane; c < a.subs; c += 64) add(part[c]);
  for (int d = 32; d; d >>= 1) best = min(best, __shfl_xor(best, d, 64));
  return {wave_sum64(z), m, m == -INFINITY ? -1 : best};
}

// A workgroup per node, a wave each for its target row, its draft row, and its token's
// probabilities in the two rows of its parent.
template <typename T>
__global__ __launch_bounds__(256) void verify_merge_kernel(VerifyArgs a) {
  const int n = blockIdx.x, lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int up = uniform(a.parents[n]), x = uniform(a.tokens[n]);
  const Tree t = tree_with(a, n);
  if (t.seq < 0) return;
  const float temp = a.temps[t.seq];
  if (w > 0 && greedy(temp)) return;
  const double rate = greedy(temp) ? 0. : rate_of(temp);
  if (w < 2) {
    if (w == 1 && (!a.draft || children_of(a, t, n - t.first) == 0)) return;
    const int row = w ? a.num_nodes + n : n;
    const RowStat mine = merge(a, row, rate);
    if (lane == 0) a.stat[row] = mine;
    return;
  }
  if (n == t.first || up < 0 || up >= n - t.first) return;
  const int parent = t.first + up;
  double* chance = reinterpret_cast<double*>(a.chance + n) + (w - 2);
  const void* logits = w == 2 ? a.logits : a.draft;
  if (!logits) {
    if (lane == 0) *chance = 1.;
    return;
  }
  const float l = static_cast<unsigned>(x) < static_cast<unsigned>(a.vocab) ? Row<T>(a, logits, parent).token(x) : -INFINITY;
  const Exp2 boost;
  const RowStat all = merge(a, w == 2 ? parent : a.num_nodes + parent, rate);
  if (lane == 0) *chance = all.z > 0. ? boost(l, all.m, rate) / all.z : 0.;
}

// R_j of a row from its parts (one wave, every lane returns it).
__device__ __forceinline__ double mass_of(const VerifyArgs& a, int j, int n) {
  if (j == 0) return 1.;
  double r = 0.;
  const double* part = a.mass + (static_cast<long long>(j - 1) * a.num_nodes + n) * a.subs;
  for (int c = threadIdx.x & 63; c < a.subs; c += 64) r += part[c];
  return wave_sum64(r);
}

// 1 less the probability of a token tried is off by 2^-53, at this size by 2^-45 of itself.
constexpr double kCoarse = 0x1p-8;

// What is left below this counts as nothing: its inverse may not be a number.
constexpr double kLeast = 0x1p-1022;

// p -> w_steps, steps >= 1; lane i has 1 / R_i (R_0 is 1).
template <int N>
__device__ __forceinline__ void take_off(double (&w)[N], const double (&q)[N], double inv, int steps) {
#pragma clang fp contract(off)  // p - q of equal rows is nothing at all
#pragma unroll
  for (int e = 0; e < N; ++e) w[e] = fmax(w[e] - q[e], 0.);
#pragma unroll 1
  for (int i = 1; i < steps; ++i) {
    const double v = lane64(inv, i);
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = fmax(fma(w[e], v, -q[e]), 0.);
  }
}

// Whether child j is accepted: its number, its token's p and q, 1 / R_i in lane i < j, 1 / R_j.
__device__ __forceinline__ bool passes(float u, double2 chance, double inv, int j, double v) {
  double w[1] = {chance.x};
  if (j) take_off(w, {chance.y}, inv, j);
  return u * chance.y < w[0] * v;
}

// The weight of a token of row n after `steps` children were taken off.
struct Weigh {
  double kp, kq, rate;  // 1 / sum of p's and of q's exponentials
  float mp, mq;
  int steps;
  double inv;  // lane i: 1 / R_i
  Exp2 boost;
  template <int N>
  __device__ __forceinline__ void operator()(const float (&lp)[N], const float (&lq)[N], double (&out)[N]) const {
#pragma clang fp contract(off)  // both rows are rounded alike
    boost(lp, mp, rate, out);
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] *= kp;
    if (steps) {
      double q[N];
      boost(lq, mq, rate, q);
#pragma unroll
      for (int e = 0; e < N; ++e) q[e] *= kq;
      take_off(out, q, inv, steps);
    }
  }
};
__device__ __forceinline__ Weigh weigh(const VerifyArgs& a, int n, int steps, double inv, float temp) {
  const RowStat p = a.stat[n];
  Weigh w = {0., 0., rate_of(temp), 0.f, 0.f, uniform(steps), inv};
  if (p.z > 0.) {
    w.kp = 1. / p.z;
    w.mp = p.m;
  }
  if (steps) {
    const RowStat q = a.stat[a.num_nodes + n];
    if (q.z > 0.) {
      w.kq = 1. / q.z;
      w.mq = q.m;
    }
  }
  return w;
}

// The weights of N places from x on of a row whose place `shift` is token 0: of its
// target's logits and, where the drafter counts, the draft's; `gone` tokens have none.
template <int N>
__device__ __forceinline__ void weights(const Weigh& w, const float (&lp)[N], const float (&lq)[N], int x, int shift, const int* gone, int num_gone, double (&out)[N]) {
  float p[N], q[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    p[e] = logit(lp[e]);
    q[e] = logit(lq[e]);
  }
  for (int k = 0; k < num_gone; ++k) {
    const int at = gone[k] + shift - x;
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = at == e ? -INFINITY : p[e];
  }
  w(p, q, out);
}

// Child j of node i of a tree, -1 where it has fewer (a wave).
__device__ __forceinline__ int child_of(const VerifyArgs& a, const Tree& t, int i, int j) {
  for (int c0 = i + 1; c0 < t.nodes; c0 += 64) {
    const int c = c0 + (threadIdx.x & 63);
    unsigned long long kids = __ballot(c < t.nodes && a.parents[t.first + min(c, t.nodes - 1)] == i);
    for (; kids && j; --j) kids &= kids - 1;
    if (kids) return c0 + __ffsll(kids) - 1;
  }
  return -1;
}

// R_j's part of kSub places (a wave), for rows with more than j children of which the
// first j are not accepted, wherever the walk may go: that a child is, the row's own
// numbers say. The logits are on their way while the rest is looked up.
template <typename T>
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs a, int j) {
  const int lane = threadIdx.x & 63, id = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int n = id / a.subs, sub = id - n * a.subs;
  if (n >= a.num_nodes) return;
  const Tree t = tree_with(a, n);
  if (t.seq < 0) return;
  const float temp = a.temps[t.seq];
  if (greedy(temp) || children_of(a, t, n - t.first) <= j) return;
  const Row<T> rp(a, a.logits, n), rq(a, a.draft, n);
  typename Row<T>::template Vec<kVec<T>> vp[kVecs<T>], vq[kVecs<T>];
#pragma unroll
  for (int i = 0; i < kVecs<T>; ++i) {
    vp[i] = rp.template fetch<kVec<T>>(place<T>(sub, i));
    vq[i] = rq.template fetch<kVec<T>>(place<T>(sub, i));
  }
  double inv = lane < j - 1 ? a.scale[static_cast<long long>(lane) * a.num_nodes + n] : 0.;
  const double v = 1. / mass_of(a, j - 1, n);
  const int kid = t.first + child_of(a, t, n - t.first, j - 1);
  const bool over = (j > 1 && lane64(inv, j - 2) < 0.) || passes(a.accept[kid], a.chance[kid], inv, j - 1, v);
  if (sub == 0 && lane == 0) a.scale[static_cast<long long>(j - 1) * a.num_nodes + n] = over ? -1. : v;
  if (over) return;
  if (lane == j - 1) inv = v;
  const Weigh w = weigh(a, n, j, inv, temp);
  const bool inside = rp.inside(sub * kSub, kSub);
  double sum = 0.;
#pragma unroll
  for (int i = 0; i < kVecs<T>; ++i) {
    float lp[kVec<T>], lq[kVec<T>];
    double x[kVec<T>];
    rp.expand(place<T>(sub, i), vp[i], inside, lp);
    rq.expand(place<T>(sub, i), vq[i], inside, lq);
    weights(w, lp, lq, 0, 0, nullptr, 0, x);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) sum += x[e];
  }
  sum = wave_sum64(sum);
  if (lane == 0) a.mass[(static_cast<long long>(j - 1) * a.num_nodes + n) * a.subs + sub] = sum;
}

// What the tokens tried leave of row n's p (one wave): the parts' sums, those that hold one of
// the tokens made anew without them.
template <typename T>
__device__ double rest_of(const VerifyArgs& a, int n, double rate, const int* gone, int num_gone) {
  const int lane = threadIdx.x & 63;
  const RowStat all = a.stat[n];
  const RowStat* part = a.part + static_cast<long long>(n) * a.subs;
  const Row<T> r(a, a.logits, n);
  const Exp2 boost;
  auto part_of = [&](int k) {  // -1: no token of the row
    const int x = uniform(gone[k]);
    return static_cast<unsigned>(x) < static_cast<unsigned>(a.vocab) ? (x + r.shift) / kSub : -1;
  };
  double sum = 0.;
#pragma unroll 1
  for (int c = lane; c < a.subs; c += 64) {
    const RowStat p = part[c];
    bool whole = p.z > 0.;
    for (int k = 0; k < num_gone; ++k) whole &= part_of(k) != c;
    sum += whole ? p.z * boost(p.m, all.m, rate) : 0.;
  }
#pragma unroll 1
  for (int k = 0; k < num_gone; ++k) {
    const int c = part_of(k);
    bool again = c < 0;
    for (int e = 0; e < k; ++e) again |= part_of(e) == c;
    if (again) continue;
    const bool inside = r.inside(c * kSub, kSub);
#pragma unroll 1
    for (int i = 0; i < kVecs<T>; ++i) {
      const int at = place<T>(c, i);
      float l[kVec<T>];
      double y[kVec<T>];
      r.expand(at, r.template fetch<kVec<T>>(at), inside, l);
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e) l[e] = logit(l[e]);
      for (int x = 0; x < num_gone; ++x) {
        const int hit = gone[x] + r.shift - at;
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e) l[e] = hit == e ? -INFINITY : l[e];
      }
      boost(l, all.m, rate, y);
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e) sum += y[e];
    }
  }
  return wave_sum64(sum) / all.z;
}

// Down a tree: which rows are accepted, and what the next token is drawn from (one
// wave, the same result in every workgroup that asks). `write`: keeps the accepted
// rows and the tokens that were not accepted at the last one. `inv`: lane i gets 1 / R_i
// there. Lanes hold 64 nodes at a time: one round trip for them, not one for each.
template <typename T>
__device__ Choice walk(const VerifyArgs& a, const Tree& t, float temp, bool write, int* gone, double& inv) {
  const int lane = threadIdx.x & 63;
  Choice r = {-1, 0, 0, 0};
  if (t.nodes == 0) return r;
  const bool top = greedy(temp);
  int at = -1, best = -1;  // the current node within the tree; its likeliest token
  double left = 1.;        // without draft logits: what the tokens tried leave of p; with them, 1 / R of the next child's test
  bool due = false;        // the tokens tried have nearly all of p: what they leave is summed for the next child
  auto reach = [&](int i, int likeliest) {
    at = i;
    best = likeliest;
    if (write && lane == 0) a.path[t.first + r.count] = t.first + i;
    r.count += 1;
    r.tried = r.steps = 0;
    left = 1.;
    due = false;
  };
  for (int i0 = 0; i0 < t.nodes; i0 += 64) {
    const int i = min(i0 + lane, t.nodes - 1), n = t.first + i;
    const int up = i0 + lane < t.nodes ? a.parents[n] : -1, token = a.tokens[n];
    const float u = a.accept[n];
    const int likeliest = top ? a.stat[n].best : -1;
    const double2 chance = top ? make_double2(0., 0.) : a.chance[n];
    if (i0 == 0) reach(0, __builtin_amdgcn_readlane(likeliest, 0));
    int from = max(i0, 1);
    while (true) {  // the next child of the current node
      const unsigned long long kids = __ballot(up == at && i0 + lane >= from);
      if (!kids) break;
      const int k = __ffsll(kids) - 1;
      from = i0 + k + 1;
      if (r.tried >= a.max_children) continue;
      if (a.draft && !top && r.tried) {  // summed, as the node has more children than were tried
        const double sum = mass_of(a, r.tried, t.first + at);
        if (!(sum >= kLeast)) {  // nothing is left to accept
          r.tried = a.max_children;
          continue;
        }
        left = 1. / sum;
      }
      if (due) left = rest_of<T>(a, t.first + at, rate_of(temp), gone, r.tried);
      due = false;
      const int x = __builtin_amdgcn_readlane(token, k);
      bool yes;
      if (top) {
        yes = best >= 0 && best == x;
      } else {
        const double pc = lane64(chance.x, k), qc = lane64(chance.y, k), uk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, u), k));
        if (a.draft) {
          yes = passes(uk, make_double2(pc, qc), inv, r.steps, left);
        } else {  // its token may have been tried before
          bool again = false;
          for (int e = 0; e < r.tried; ++e) again |= gone[e] == x;
          yes = !again && uk < pc / left;
          if (!yes && !again) {
            left -= pc;
            due = pc > 0. && left < kCoarse;
          }
        }
      }
      if (yes) {
        reach(i0 + k, __builtin_amdgcn_readlane(likeliest, k));
      } else {
        if (lane == 0) gone[r.tried] = x;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes read it
        __builtin_amdgcn_wave_barrier();
        r.tried += 1;
        if (a.draft && !top) {
          if (lane == r.steps) inv = left;
          r.steps += 1;
        }
      }
    }
  }
  r.node = t.first + at;
  return r;
}

// Sequence s's walk, and a part of the sum that its next token is drawn by.
template <typename T>
__global__ __launch_bounds__(256) void verify_walk_kernel(VerifyArgs a) {
  __shared__ Choice sr;
  __shared__ int gone[64];
  __shared__ double scales[64];
  const int groups = a.subs / 4, s = blockIdx.x / groups, c = blockIdx.x - s * groups;
  const int sub = 4 * c + uniform(threadIdx.x >> 6);
  const Tree t = tree_of(a, s);
  const float temp = a.temps[s];
  if (threadIdx.x < 64) {
    double inv = 0.;
    const Choice r = walk<T>(a, t, temp, c == 0, gone, inv);
    scales[threadIdx.x] = inv;
    if (threadIdx.x == 0) {
      sr = r;
      if (c == 0) a.choice[s] = r;
    }
  }
  __syncthreads();
  const Choice r = sr;
  if (r.node < 0 || greedy(temp)) return;
  const Row<T> rp(a, a.logits, r.node), rq(a, r.steps ? a.draft : a.logits, r.node);
  const bool inside = rp.inside(sub * kSub, kSub);
  typename Row<T>::template Vec<kVec<T>> vp[kVecs<T>], vq[kVecs<T>];
#pragma unroll
  for (int i = 0; i < kVecs<T>; ++i) {
    vp[i] = rp.template fetch<kVec<T>>(place<T>(sub, i));
    vq[i] = rq.template fetch<kVec<T>>(place<T>(sub, i));  // where no drafter counts, the same again
  }
  const int num_gone = a.draft ? 0 : r.tried;
  if (c == 0 && static_cast<int>(threadIdx.x) < num_gone) a.tried[s * a.max_children + threadIdx.x] = gone[threadIdx.x];
  if (c == 0 && static_cast<int>(threadIdx.x) < r.steps) a.last[s * a.max_children + threadIdx.x] = scales[threadIdx.x];
  const Weigh w = weigh(a, r.node, r.steps, scales[threadIdx.x & 63], temp);
  double sum = 0.;
#pragma unroll
  for (int i = 0; i < kVecs<T>; ++i) {
    double x[kVec<T>];
    float lp[kVec<T>], lq[kVec<T>];
    rp.expand(place<T>(sub, i), vp[i], inside, lp);
    rq.expand(place<T>(sub, i), vq[i], inside, lq);
    weights(w, lp, lq, place<T>(sub, i), rp.shift, gone, num_gone, x);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) sum += x[e];
  }
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) a.weight[static_cast<long long>(s) * a.subs + sub] = sum;
}

// N numbers of each thread, in the threads' order: run[i] is the sum of all up to and
// with its i-th. Returns the sum of all. Every thread calls it.
template <int N>
__device__ __forceinline__ double block_scan(const double (&x)[N], double (&run)[N], double* tmp) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double mine = 0.;
#pragma unroll
  for (int i = 0; i < N; ++i) mine += x[i];
  const double incl = wave_scan64(mine);
  __syncthreads();  // tmp is free
  if (lane == 63) tmp[w] = incl;
  __syncthreads();
  double before = 0., all = 0.;
  for (int i = 0; i < 4; ++i) {
    if (i < w) before += tmp[i];
    all += tmp[i];
  }
  before += dpp64<0x138>(incl);  // of the lanes before this one (wave_shr 1)
#pragma unroll
  for (int i = 0; i < N; ++i) run[i] = before += x[i];
  return all;
}

// One workgroup per sequence: its rows' place in the result, and its next token.
template <typename T>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs a) {
  constexpr int kParts = 5;  // of a row, to a thread
  static_assert(((1 << 20) / kWalk + 1) * (kWalk / kSub) <= kParts * 256, "the largest vocabulary's");
  __shared__ int counts[8], found[4], last[4];
  __shared__ double tmp[4], start;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  double x[kParts], run[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) x[i] = tid * kParts + i < a.subs ? a.weight[static_cast<long long>(s) * a.subs + tid * kParts + i] : 0.;
  Choice r = a.choice[s];
  const Tree t = tree_of(a, s);
  const float temp = a.temps[s], u = a.sample[s];
  int b = 0, n = 0;
  for (int i = tid; i < a.num_seqs; i += 256) {
    const int count = a.choice[i].count;
    n += count;
    if (i < s) b += count;
  }
  for (int d = 32; d; d >>= 1) {
    n += __shfl_xor(n, d, 64);
    b += __shfl_xor(b, d, 64);
  }
  if (lane == 0) {
    counts[wave] = b;
    counts[4 + wave] = n;
  }
  __syncthreads();
  const int before = counts[0] + counts[1] + counts[2] + counts[3], total = counts[4] + counts[5] + counts[6] + counts[7];
  for (int i = tid; i < r.count && before + i < a.num_nodes; i += 256) a.rows[before + i] = a.path[t.first + i];
  for (long long i = total + s * 256LL + tid; i < a.num_nodes; i += a.num_seqs * 256LL) a.rows[i] = -1;
  if (tid == 0) {
    a.row_starts[s] = before;
    if (s == a.num_seqs - 1) a.row_starts[a.num_seqs] = total;
  }
  if (r.node < 0 || greedy(temp)) {
    if (tid == 0) a.next[s] = r.node < 0 ? -1 : a.stat[r.node].best;
    return;
  }
  // The part of the row in which the sum passes u times all.
  int num_gone = a.draft ? 0 : r.tried;
  double sum = block_scan(x, run, tmp);
  if (!(sum > 0.)) {  // nothing is left of p: p itself
    const RowStat all = a.stat[r.node];
    r.steps = 0;
    num_gone = 0;
    const Exp2 boost;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int c = tid * kParts + i;
      const RowStat part = a.part[static_cast<long long>(r.node) * a.subs + min(c, a.subs - 1)];
      x[i] = c < a.subs && part.z > 0. ? part.z * boost(part.m, all.m, rate_of(temp)) / all.z : 0.;
    }
    sum = block_scan(x, run, tmp);
  }
  const double goal = u * sum;
  // The first of all threads' numbers that has a weight and at which the sum is past the
  // goal, else the last one with a weight, else -1. Numbers ascend with the threads.
  int hit = INT_MAX, end = -1;
  auto note = [&](int number, double weight, double upto) {
    if (weight > 0.) {
      if (upto > goal && hit == INT_MAX) hit = number;
      end = number;
    }
  };
  auto first = [&] {
    const unsigned long long hits = __ballot(hit != INT_MAX), ends = __ballot(end >= 0);
    const int h = __shfl(hit, hits ? __ffsll(hits) - 1 : 0, 64), e = __shfl(end, ends ? 63 - __clzll(ends) : 0, 64);
    __syncthreads();
    if (lane == 0) {
      found[wave] = h;
      last[wave] = e;
    }
    __syncthreads();
    hit = INT_MAX;
    end = -1;
    const int f = min(min(found[0], found[1]), min(found[2], found[3]));
    return f != INT_MAX ? f : max(max(last[0], last[1]), max(last[2], last[3]));
  };
#pragma unroll
  for (int i = 0; i < kParts; ++i) note(tid * kParts + i, x[i], run[i]);
  const int part = first();
  if (part < 0) {
    if (tid == 0) a.next[s] = -1;
    return;
  }
#pragma unroll
  for (int i = 0; i < kParts; ++i)
    if (tid * kParts + i == part) start = run[i] - x[i];
  __syncthreads();
  // And the token there.
  const Weigh w = weigh(a, r.node, r.steps, lane < r.steps ? a.last[s * a.max_children + lane] : 0., temp);
  const Row<T> rp(a, a.logits, r.node), rq(a, r.steps ? a.draft : a.logits, r.node);
  const int p0 = part * kSub;
  double y[4], upto[4];
  float lp[4], lq[4];
  rp.expand(p0 + tid * 4, rp.template fetch<4>(p0 + tid * 4), rp.inside(p0, kSub), lp);
  rq.expand(p0 + tid * 4, rq.template fetch<4>(p0 + tid * 4), rp.inside(p0, kSub), lq);
  weights(w, lp, lq, p0 + tid * 4, rp.shift, a.tried + s * a.max_children, num_gone, y);
  block_scan(y, upto, tmp);
#pragma unroll
  for (int i = 0; i < 4; ++i) note(p0 + tid * 4 + i, y[i], start + upto[i]);
  const int at = first();
  if (tid == 0) a.next[s] = at < 0 ? -1 : at - rp.shift;
}

// Parts of a row (places are counted from up to 7 elements before it), in whole fours.
int subs_of(int vocab) { return (vocab + 7 + kWalk - 1) / kWalk * 4; }

const char* check_shape(int vocab, int num_seqs, int num_nodes, int max_nodes, int max_children) {
  if (vocab < 1 || vocab > (1 << 20)) return "vocab outside [1, 2^20]";
  if (num_seqs < 1 || num_seqs > kMaxSeqs) return "num_seqs outside [1, 8192]";
  if (num_nodes < 1 || num_nodes > (1 << 20)) return "num_nodes outside [1, 2^20]";
  if (max_nodes < 1 || max_nodes > kMaxNodes) return "max_nodes outside [1, 1024]";
  if (max_children < 1 || max_children > 64) return "max_children outside [1, 64]";
  // a launch has less than 2^32 threads
  if (num_nodes * (subs_of(vocab) / 4LL) >= (1LL << 23)) return "num_nodes * vocab: ceil((vocab + 7) / 4096) times num_nodes must be below 2^23";
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
  take(a.part, rows * a.subs);
  take(a.stat, rows);
  take(a.chance, a.num_nodes);
  take(a.choice, a.num_seqs);
  take(a.weight, static_cast<long long>(a.num_seqs) * a.subs);
  take(a.path, a.num_nodes);
  take(a.tried, static_cast<long long>(a.num_seqs) * a.max_children);
  take(a.last, draft ? static_cast<long long>(a.num_seqs) * a.max_children : 0);
  const long long sums = draft ? static_cast<long long>(a.max_children - 1) * a.num_nodes : 0;
  take(a.scale, sums);
  take(a.mass, sums * a.subs);
  return at;
}

template <typename T>
void launch(const VerifyArgs& a, hipStream_t s) {
  auto waves = [](long long n) { return dim3(static_cast<unsigned>((n + 3) / 4)); };  // in workgroups of four
  const dim3 stats = waves((a.draft ? 2LL : 1LL) * a.num_nodes * a.subs), mass = waves(static_cast<long long>(a.num_nodes) * a.subs);
  IRON_LAUNCH((verify_stats_kernel<T>), stats, dim3(256), 0, s, a);
  IRON_LAUNCH((verify_merge_kernel<T>), dim3(a.num_nodes), dim3(256), 0, s, a);
  if (a.draft)
    for (int j = 1; j < a.max_children; ++j) IRON_LAUNCH((verify_mass_kernel<T>), mass, dim3(256), 0, s, a, j);
  IRON_LAUNCH((verify_walk_kernel<T>), dim3(a.num_seqs * (a.subs / 4)), dim3(256), 0, s, a);
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
  a.subs = subs_of(vocab);
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
  // The last launch reads while it writes the results, so these and the workspace lie apart from all else.
  const long long elements = static_cast<long long>(num_nodes) * vocab * (dtype == 2 ? 4 : 2);
  const struct {
    const void* at;
    long long bytes;
  } spans[] = {{rows, 4LL * num_nodes}, {row_starts, 4LL * (num_seqs + 1)}, {next_tokens, 4LL * num_seqs}, {workspace, need},
               {logits, elements}, {draft_logits, draft_logits ? elements : 0}, {tokens, 4LL * num_nodes}, {parents, 4LL * num_nodes},
               {node_starts, 4LL * (num_seqs + 1)}, {temperatures, 4LL * num_seqs}, {accept_draws, 4LL * num_nodes}, {sample_draws, 4LL * num_seqs}};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 12; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(spans[i].at), y = reinterpret_cast<uintptr_t>(spans[j].at);
      IRON_REQUIRE(x + spans[i].bytes <= y || y + spans[j].bytes <= x || !spans[j].bytes,
                   "%s: rows, row_starts, next_tokens and the workspace must not overlap each other or an input", who);
    }
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
  a.subs = subs_of(vocab);
  lay_out(a, draft_logits != nullptr, static_cast<char*>(workspace));
  hipStream_t s = static_cast<hipStream_t>(stream);
  dtype == 0 ? launch<uint16_t>(a, s) : dtype == 1 ? launch<_Float16>(a, s) : launch<float>(a, s);
  return check_launch("draft_verify");
}
