// Draft trees for gfx950: the tree's masks, the verification of its tokens
// against the target model, and the move of the accepted path's K and V.
//
// A tree of N nodes is given by parents: node 0 is the last token of the
// sequence (parent -1), every other node comes after its parent; a parent
// below -1 marks a padding slot.
#include <type_traits>

#include "kernels.hpp"

namespace cie {

// ---- masks -----------------------------------------------------------------
//
// One workgroup per sequence, one thread per node. A parent's index is below
// its child's, so the walk to the root meets the ancestors in falling order:
// the row's words are finished one after another, and every walk ends. A thread
// walks twice, for the depth and validity and for the bits: two dependent LDS reads
// a level of the tree, 0.19 us. Trees of a few levels 1.7-1.9 us up to 128 nodes,
// the time of an empty launch, and 5 and 18 for 512 and 1024 nodes, whose threads
// each write a row of their own; a chain of 26 nodes 5.3, of 128 23, of 1024 194.
__global__ __launch_bounds__(1024) void draft_mask_kernel(const int32_t* parents, int32_t* mask, int32_t* depths,
                                                         uint32_t* status, int N, int W) {
  __shared__ int32_t par[kTreeMaxNodes];
  const int b = blockIdx.x, i = threadIdx.x;
  if (i < N) par[i] = parents[(int64_t)b * N + i];
  __syncthreads();
  if (i >= N) return;
  // depth of a node, -1 for padding, -2 for a node whose chain is broken
  // (a parent that does not come before its child, or is padding)
  int depth = par[i] < -1 ? -1 : 0;
  for (int at = i; depth >= 0 && par[at] != -1; ++depth) {
    const int up = par[at];
    if (up >= at || up < -1) {
      depth = -2;
      break;
    }
    at = up;
  }
  depths[(int64_t)b * N + i] = depth;
  if (depth == -2 && status) atomicOr(status, 1u);
  int32_t* row = mask + ((int64_t)b * N + i) * W;
  for (int w = depth < 0 ? 0 : (i >> 5) + 1; w < W; ++w) row[w] = 0;
  if (depth < 0) return;
  int w = i >> 5;
  uint32_t bits = 0;
  for (int at = i; at >= 0; at = par[at]) {
    for (; w > at >> 5; --w) {
      row[w] = (int32_t)bits;
      bits = 0;
    }
    bits |= 1u << (at & 31);
  }
  for (; w >= 0; --w) {
    row[w] = (int32_t)bits;
    bits = 0;
  }
}

hipError_t launch_draft_masks(const int32_t* parents, int32_t* mask, int32_t* depths, uint32_t* status, int B, int N,
                              hipStream_t stream) {
  hipLaunchKernelGGL(draft_mask_kernel, dim3((unsigned)B), dim3((unsigned)((N + 63) / 64 * 64)), 0, stream, parents,
                     mask, depths, status, N, (N + 31) / 32);
  return hipGetLastError();
}

// ---- verification ------------------------------------------------------------
//
// The walk from node 0. At node a with target probabilities p and draft
// probabilities q, the children are tried in order; child i with token x is
// accepted iff
//   u_i q(x) < p(x)      (q(x) = 1 when the drafts are the draft's own picks)
// and after a rejection
//   p <- max(p - q, 0) / its sum      (p without x, over its sum)
//   q <- q without x, over its sum    (drafts without replacement)
// each only if that sum is over 2^-40. When no child is accepted the last token
// is the first y with p(0) + .. + p(y) > u_0 (p's sum).
//
// The residual after some rejections needs no copy of p: it is max(p - c q, 0) / W
// for running scalars, c <- c + W / S and W <- sum max(p - c q, 0), S the sum
// of what is left of q; a token that q has lost keeps the p it had then. One
// pass over the rows per rejection gives W (one per node for the draft's own
// picks, whose W follows from the children's p), and none is needed before a
// first rejection: each child's p(x), q(x) and u are fetched once for the whole
// tree, one thread a node, and with them whether the child passes if it is the
// first one tried.
//
// All sums are 64-bit: the last token is a comparison of a sum over the
// vocabulary with u_0 times that sum, and has to come out the same whatever the
// order of the summation; in 32 bits one draw in some thousands would not.
//
// The vocabulary is cut into 64 parts at most whose sums are kept, so that the
// part holding the last token follows from them and only it is read again.
//
// One workgroup per sequence: start 1-1.5 us, a step down the tree 0.1, the last
// token 2.8, and the passes, at what one CU reads (wave_sums), one after another and
// with the other CUs idle where sequences are few. Over 128000 fp32 tokens a call
// without a rejection takes 11 us whatever the batch; each rejection adds 10 (with
// replacement) or 13 (without), the first one some 10 more for a draft's own picks
// and 2 for every other: one sequence with eight rejections at a node 97, 127 and 34.
// 8 chains of 5 over 32000 tokens 8-10 us, most of it one pass of p; 32 trees of 26
// over 128000 44-57, the sequence with three rejections at a node. (Summing every row
// with the whole GPU beforehand, for c = 1: 63 -> 150 us there, 16.6 -> 20 for the
// chains: the walk needs few of them. Only the rows of nodes whose first child fails
// are needed, which the gathered p, q and u tell; not built.)
constexpr int kVerifyWaves = 16, kVerifyThreads = 64 * kVerifyWaves;
constexpr int kParts = 64;
constexpr double kNoMass = 0x1p-40;

template <int DT> struct ProbElt;  // 0 fp16, 1 bf16, 2 fp32: 16 bytes a load, rows of any alignment
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x4 u32x4_4 __attribute__((aligned(4)));
__device__ __forceinline__ u32x4 load_part16(const uint16_t* p, int n) {
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  return v;
}
__device__ __forceinline__ void clear16(u32x4& v, int e) {
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] &= d != e >> 1 ? 0xffffffffu : e & 1 ? 0xffffu : 0xffff0000u;
}
template <> struct ProbElt<2> {
  typedef float T;
  static constexpr int V = 4;
  static __device__ __forceinline__ float at(const T* p) { return *p; }
  static __device__ __forceinline__ u32x4 load(const T* p) { return *reinterpret_cast<const u32x4_4*>(p); }
  static __device__ __forceinline__ float get(u32x4 v, int e) { return __uint_as_float(v[e]); }
  // the first n elements, then zeros; element e cleared
  static __device__ __forceinline__ u32x4 load_part(const T* p, int n) {
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) v[e] = __float_as_uint(p[e]);
    return v;
  }
  static __device__ __forceinline__ void clear(u32x4& v, int e) {
#pragma unroll
    for (int d = 0; d < 4; ++d) v[d] = d == e ? 0u : v[d];
  }
};
template <> struct ProbElt<1> {
  typedef uint16_t T;
  static constexpr int V = 8;
  static __device__ __forceinline__ float at(const T* p) { return __uint_as_float((uint32_t)*p << 16); }
  static __device__ __forceinline__ u32x4 load(const T* p) { return *reinterpret_cast<const u32x4_any*>(p); }
  static __device__ __forceinline__ float get(u32x4 v, int e) {
    return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
  }
  static __device__ __forceinline__ u32x4 load_part(const T* p, int n) { return load_part16(p, n); }
  static __device__ __forceinline__ void clear(u32x4& v, int e) { clear16(v, e); }
};
template <> struct ProbElt<0> {
  typedef uint16_t T;
  static constexpr int V = 8;
  static __device__ __forceinline__ float at(const T* p) { return (float)__builtin_bit_cast(_Float16, *p); }
  static __device__ __forceinline__ u32x4 load(const T* p) { return *reinterpret_cast<const u32x4_any*>(p); }
  static __device__ __forceinline__ float get(u32x4 v, int e) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? v[e >> 1] >> 16 : v[e >> 1]));
  }
  static __device__ __forceinline__ u32x4 load_part(const T* p, int n) { return load_part16(p, n); }
  static __device__ __forceinline__ void clear(u32x4& v, int e) { clear16(v, e); }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Children of node `cur` after node `after`: the next one (with token x, if `tok`
// is given), or -1; every wave finds it for itself.
__device__ __forceinline__ int next_child(const int32_t* par, int N, int cur, int after, int lane,
                                          const int32_t* tok = nullptr, int x = 0) {
  for (int c = (after + 1) >> 6; 64 * c < N; ++c) {
    const int i = 64 * c + lane;
    const uint64_t m =
        __builtin_amdgcn_ballot_w64(i < N && i > after && par[i] == cur && (!tok || tok[i] == x));
    if (m) return 64 * c + __builtin_ctzll(m);
  }
  return -1;
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[i] : (int64_t)static_cast<const int32_t*>(tokens)[i];
}
__device__ __forceinline__ void token_store(void* tokens, int bytes, int64_t i, int64_t v) {
  if (bytes == 8) static_cast<int64_t*>(tokens)[i] = v;
  else static_cast<int32_t*>(tokens)[i] = (int32_t)v;
}

// What one pass over the vocabulary sums: p, or the residual max(p - c q, 0);
// either of them without the listed tokens; that residual and q without them.
enum { kSumP, kSumPWithout, kSumRest, kSumRestWithout, kSumRestQWithout };

// Tokens of a part of the vocabulary: what one wave has in flight at once, or
// more where 64 parts of that do not cover it.
__device__ __forceinline__ int part_tokens(int V) {
  constexpr int E = 64 * 32;
  return ((V + kParts - 1) / kParts + E - 1) / E * E;
}

// Those sums for parts w, w + 16, .. of a row, by one wave, to psum[part] (and
// that of q to pq[part]). The listed tokens (the children of the node) are left
// out rather than subtracted later: what remains may be a small part of the sum.
// Bound by what one CU has under way to memory: 78 GB/s, p alone or both rows
// (128000 fp32 tokens: 6.6 and 13 us). The next block, of this part or the next,
// is asked for before this one is summed; full parts go through a loop without
// a branch around a load, the last one apart.
template <int DT, int WHAT>
__device__ __forceinline__ void wave_sums(const typename ProbElt<DT>::T* P, const typename ProbElt<DT>::T* Q, double c,
                                          int V, int w, int lane, const int32_t* list, int nlist, double* psum,
                                          double* pq) {
  using E = ProbElt<DT>;
  constexpr bool REST = WHAT >= kSumRest, LIST = WHAT != kSumP && WHAT != kSumRest;
  constexpr int U = (DT == 2 || (REST && LIST) ? 16 : 32) / E::V, BLOCK = 64 * E::V * U;  // (two blocks in 128 registers)
  struct Block {
    u32x4 a[U], q[U];
  };
  const int per = part_tokens(V), full = V / per, blocks = per / BLOCK;
  double s[2] = {0.0, 0.0}, sq = 0.0;
  auto load = [&](Block& x, int at) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int y = at + (64 * u + lane) * E::V;
      x.a[u] = E::load(P + y);
      if (REST) x.q[u] = E::load(Q + y);
    }
  };
  auto add = [&](Block& x, int at) {
    if (LIST)
      for (int g0 = 0; g0 < nlist; g0 += 64) {
        const int mine = g0 + lane < nlist ? list[g0 + lane] - at : -1;
        for (uint64_t in = __builtin_amdgcn_ballot_w64(mine >= 0 && mine < BLOCK); in; in &= in - 1) {
          const int rel = __builtin_amdgcn_readlane(mine, __builtin_ctzll(in));
          const int own = rel / E::V;  // 64 u + lane of the token's element
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (own == 64 * u + lane) {
              E::clear(x.a[u], rel % E::V);
              if (REST) E::clear(x.q[u], rel % E::V);
            }
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E::V; ++e) {
        const double pp = (double)E::get(x.a[u], e);
        if (REST) {
          const double qq = (double)E::get(x.q[u], e);
          s[e & 1] += __builtin_fmax(__builtin_fma(-c, qq, pp), 0.0);
          if (WHAT == kSumRestQWithout) sq += qq;
        } else {
          s[e & 1] += pp;
        }
      }
  };
  auto finish = [&](int part) {
    const double sum = wave_sum(s[0] + s[1]);
    const double qsum = WHAT == kSumRestQWithout ? wave_sum(sq) : 0.0;
    if (lane == 0) psum[part] = sum;
    if (WHAT == kSumRestQWithout && lane == 0) pq[part] = qsum;
    s[0] = s[1] = sq = 0.0;
  };
  if (w < full) {
    Block now, next;
    int part = w, k = 0;
    load(now, part * per);
    for (;;) {
      const int at = part * per + k * BLOCK;
      const bool ends = k + 1 == blocks;
      const int part2 = ends ? part + kVerifyWaves : part, k2 = ends ? 0 : k + 1;
      if (part2 >= full) break;
      load(next, part2 * per + k2 * BLOCK);
      add(now, at);
      if (ends) finish(part);
      now = next;
      part = part2, k = k2;
    }
    add(now, part * per + k * BLOCK);
    finish(part);
  }
  if (full * per < V && (full & (kVerifyWaves - 1)) == w) {
    for (int at = full * per; at < V; at += BLOCK) {
      Block x;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int y = at + (64 * u + lane) * E::V;
        x.a[u] = x.q[u] = u32x4{0u, 0u, 0u, 0u};
        if (y + E::V <= V) {
          x.a[u] = E::load(P + y);
          if (REST) x.q[u] = E::load(Q + y);
        } else if (y < V) {
          x.a[u] = E::load_part(P + y, V - y);
          if (REST) x.q[u] = E::load_part(Q + y, V - y);
        }
      }
      add(x, at);
    }
    finish(full);
  }
}

enum { kDraftPicks = 0, kDraftIid = 1, kDraftTree = 2 };

// A tree's parents and tokens as the kernels use them: a node that can never be
// tried (a padding slot, a parent that does not come before it, a token outside
// the vocabulary) has parent -2.
__device__ __forceinline__ void tree_node(const VerifyParams& p, int b, int i, int& up, int& x) {
  up = p.parents[(int64_t)b * p.N + i];
  const int64_t t = token_at(p.draft_tokens, p.token_bytes, (int64_t)b * p.N + i);
  const bool known = t >= 0 && t < p.V;
  x = known ? (int)t : -1;
  if (i > 0 && !(up >= 0 && up < i && known)) up = -2;
}

template <int DT, int MODE>
__global__ __launch_bounds__(kVerifyThreads) void verify_draft_kernel(const VerifyParams p) {
  using E = ProbElt<DT>;
  using T = typename E::T;
  __shared__ int32_t par[kTreeMaxNodes], tok[kTreeMaxNodes], path[kTreeMaxNodes];
  __shared__ int32_t list[kTreeMaxNodes];                  // the distinct tokens of the node's children
  __shared__ uint8_t out_of[kVerifyWaves][kTreeMaxNodes];  // which of them are out, each wave's own copy
  __shared__ float pg[kTreeMaxNodes], qg[kTreeMaxNodes], lp[kTreeMaxNodes], lq[kTreeMaxNodes];
  __shared__ double kept[kTreeMaxNodes];  // drafts without replacement: what p has left of a token that q lost
  __shared__ double ug[kTreeMaxNodes];
  __shared__ double psum[2][kParts], pq[kParts], wpre[kVerifyWaves];
  __shared__ int32_t first_of[kTreeMaxNodes];  // a node's first child
  __shared__ uint8_t easy[kTreeMaxNodes];      // accepted if nothing was rejected before it
  __shared__ int found, lastpos;
  const int b = blockIdx.x, i = threadIdx.x, lane = i & 63;
  const int w = __builtin_amdgcn_readfirstlane(i >> 6);
  const int N = p.N, V = p.V;
  if (i < N) first_of[i] = N;
  __syncthreads();
  const T* const target = static_cast<const T*>(p.target) + (int64_t)b * p.ts0;
  const T* const draft = MODE == kDraftPicks ? nullptr : static_cast<const T*>(p.draft) + (int64_t)b * p.ds0;
  if (i < N) {
    int up, x;
    tree_node(p, b, i, up, x);
    const bool child = i > 0 && up >= 0;
    par[i] = up;
    tok[i] = x;
    pg[i] = child ? E::at(target + (int64_t)up * p.ts1 + x) : 0.f;
    qg[i] = child && MODE != kDraftPicks ? E::at(draft + (int64_t)up * p.ds1 + x) : 1.f;
    ug[i] = p.uniform_bytes == 8 ? static_cast<const double*>(p.uniforms)[(int64_t)b * N + i]
                                 : (double)static_cast<const float*>(p.uniforms)[(int64_t)b * N + i];
    const double r = MODE == kDraftPicks ? (double)pg[i] : __builtin_fmax((double)pg[i], 0.0);
    easy[i] = child && ug[i] * (double)qg[i] < r;
    if (child) atomicMin(&first_of[up], i);
  }
  if (i == 0) found = V, lastpos = -1;
  __syncthreads();
  const bool active = par[0] == -1;  // a padding slot at node 0: no sequence here
  int cur = 0, count = active ? 1 : 0;
  int64_t last = -1;
  if (active) {
    const int per = part_tokens(V), parts = (V + per - 1) / per;
    const T *P = nullptr, *Q = nullptr;
    int buf = 0;   // psum[buf] holds the sums of the current residual's parts when `have`
    int nlist = 0;
    bool have = false;
    double qlist = 0.0;  // sum of q without the listed tokens
    // One pass over the row. The parts' sums go to psum[buf ^ 1], the total is the
    // same on every thread.
    auto scan = [&](auto what, double cc) {
      constexpr int WHAT = decltype(what)::value;
      wave_sums<DT, WHAT>(P, Q, cc, V, w, lane, list, nlist, psum[buf ^ 1], pq);
      __syncthreads();
      const double t = wave_sum(lane < parts ? psum[buf ^ 1][lane] : 0.0);
      if (WHAT == kSumRestQWithout) qlist = wave_sum(lane < parts ? pq[lane] : 0.0);
      __syncthreads();  // pq and the other buffer may be written again
      return t;
    };
    uint8_t* const gone = out_of[w];
    double W, c, S, total, rest = 0.0;
    // p's residual at listed token g for the scalar cc
    auto rest_of = [&](int g, double cc) {
      if (MODE == kDraftPicks) return gone[g] ? 0.0 : (double)lp[g];
      return gone[g] ? kept[g] : __builtin_fmax(__builtin_fma(-cc, (double)lq[g], (double)lp[g]), 0.0);
    };
    // the sum of f over the list, on every lane
    auto over_list = [&](auto f) {
      double t = 0.0;
      for (int g = lane; g < nlist; g += 64) t += f(g);
      return wave_sum(t);
    };
    // a token's place in the list, or -1
    auto place = [&](int x) {
      for (int g0 = 0; g0 < nlist; g0 += 64) {
        const uint64_t m = __builtin_amdgcn_ballot_w64(g0 + lane < nlist && list[g0 + lane] == x);
        if (m) return g0 + (int)__builtin_ctzll(m);
      }
      return -1;
    };
    for (;;) {
      if (first_of[cur] < N && easy[first_of[cur]]) {  // the common step: two reads of LDS
        cur = first_of[cur];
        if (i == 0) path[count] = cur;
        ++count;
        continue;
      }
      P = target + (int64_t)cur * p.ts1;
      if (MODE != kDraftPicks) Q = draft + (int64_t)cur * p.ds1;
      W = 1.0, c = 0.0, S = 1.0, total = 0.0, nlist = 0, have = false;
      bool first = true;  // no rejection at this node yet
      int taken = -1;
      for (int ch = first_of[cur] < N ? first_of[cur] : -1; ch >= 0; ch = next_child(par, N, cur, ch, lane)) {
        const int x = tok[ch];
        int at = MODE == kDraftIid ? -1 : place(x);
        const bool out = at >= 0 && gone[at];  // out of p (picks) or of q (no replacement)
        const double qx = (double)qg[ch];
        const double r = at >= 0                ? rest_of(at, c)
                         : MODE == kDraftPicks ? (double)pg[ch]
                                               : __builtin_fmax(__builtin_fma(-c, qx, (double)pg[ch]), 0.0);
        const double qq = MODE == kDraftPicks ? 1.0 : MODE == kDraftTree && out ? 0.0 : qx / S;
        if (ug[ch] * qq < r / W) {
          taken = ch;
          break;
        }
        if (MODE != kDraftIid && first) {
          // (every wave writes the same list; none still reads the one before)
          __syncthreads();
          for (int k = ch; k >= 0; k = next_child(par, N, cur, k, lane)) {
            if (place(tok[k]) >= 0) continue;
            list[nlist] = tok[k];
            lp[nlist] = pg[k];
            lq[nlist] = qg[k];
            gone[nlist] = 0;
            ++nlist;
          }
          at = 0;
        }
        if (MODE == kDraftPicks) {
          if (first) {
            rest = scan(std::integral_constant<int, kSumPWithout>{}, 0.0);
            buf ^= 1;
            have = true;
            total = rest + over_list([&](int g) { return rest_of(g, 0.0); });
          }
          const bool was = gone[at];
          gone[at] = 1;
          const double t = rest + over_list([&](int g) { return rest_of(g, 0.0); });
          if (t / W > kNoMass) W = total = t;
          else gone[at] = was;
        } else {
          const double c2 = c + W / S;
          double t;
          if (MODE == kDraftIid) t = scan(std::integral_constant<int, kSumRest>{}, c2);
          else if (first) t = scan(std::integral_constant<int, kSumRestQWithout>{}, c2);
          else t = scan(std::integral_constant<int, kSumRestWithout>{}, c2);
          if (MODE == kDraftTree) t += over_list([&](int g) { return rest_of(g, c2); });
          if (t / W > kNoMass) {
            c = c2;
            W = total = t;
            buf ^= 1;
            have = true;
          }
          if (MODE == kDraftTree && !out) {
            gone[at] = 1;
            const double m = qlist + over_list([&](int g) { return gone[g] ? 0.0 : (double)lq[g]; });
            if (m / S > kNoMass) {
              S = m;
              kept[at] = __builtin_fmax(__builtin_fma(-c, qx, (double)pg[ch]), 0.0);
            } else {
              gone[at] = 0;
            }
          }
        }
        first = false;
      }
      if (taken < 0) break;
      cur = taken;
      if (i == 0) path[count] = cur;
      ++count;
    }
    if (!have) {  // nothing was rejected at the last node, or nothing is left of p - q there: c is 0
      nlist = 0;
      total = scan(std::integral_constant<int, kSumP>{}, 0.0);
      buf ^= 1;
    }
    // the part that the last token lies in (the same on every wave)
    const double goal = ug[0] * total;
    double mine = lane < parts ? psum[buf][lane] : 0.0;
    if (MODE != kDraftIid)
      for (int g = 0; g < nlist; ++g) {
        const int at = list[g] - lane * per;
        if (at >= 0 && at < per) mine += rest_of(g, c);
      }
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(incl, o);
      if (lane >= o) incl += up;
    }
    const uint64_t some = __builtin_amdgcn_ballot_w64(mine > 0.0);
    const uint64_t over = __builtin_amdgcn_ballot_w64(mine > 0.0 && incl > goal);
    const int part = over ? (int)__builtin_ctzll(over) : some ? 63 - (int)__builtin_clzll(some) : -1;
    double before = __shfl(incl - mine, max(part, 0));
    // (from here nothing writes the list, and every wave's copy of `gone` says the same)
    const int plo = min(max(part, 0) * per, V), phi = part < 0 ? plo : min(plo + per, V);
    constexpr int R = 2;  // tokens of a thread at once
    for (int at = plo; at < phi; at += R * kVerifyThreads) {
      double r[R], sum = 0.0;
#pragma unroll
      for (int e = 0; e < R; ++e) {
        const int y = at + R * i + e;
        r[e] = 0.0;
        if (y < phi) {
          r[e] = (double)E::at(P + y);
          if (MODE != kDraftPicks && c != 0.0) r[e] = __builtin_fmax(__builtin_fma(-c, (double)E::at(Q + y), r[e]), 0.0);
        }
      }
      if (MODE != kDraftIid)
        for (int g = 0; g < nlist; ++g)
#pragma unroll
          for (int e = 0; e < R; ++e) r[e] = list[g] == at + R * i + e ? rest_of(g, c) : r[e];
#pragma unroll
      for (int e = 0; e < R; ++e) sum += r[e];
      double upto = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(upto, o);
        if (lane >= o) upto += up;
      }
      if (lane == 63) wpre[w] = upto;
      __syncthreads();
      double run = before + (upto - sum);
      for (int x = 0; x < kVerifyWaves; ++x) {
        if (x < w) run += wpre[x];
        before += wpre[x];
      }
      int hit = V, pos = -1;
#pragma unroll
      for (int e = R - 1; e >= 0; --e)
        if (r[e] > 0.0 && pos < 0) pos = at + R * i + e;
#pragma unroll
      for (int e = 0; e < R; ++e) {
        run += r[e];
        if (r[e] > 0.0 && run > goal && hit == V) hit = at + R * i + e;
      }
      // (one atomic a wave: 64 on one word take the LDS 64 turns)
      const uint64_t hits = __builtin_amdgcn_ballot_w64(hit < V), any = __builtin_amdgcn_ballot_w64(pos >= 0);
      if (hits && lane == (int)__builtin_ctzll(hits)) atomicMin(&found, hit);
      if (any && lane == 63 - (int)__builtin_clzll(any)) atomicMax(&lastpos, pos);
      __syncthreads();
      if (found < V) break;
    }
    last = found < V ? found : lastpos;  // (rounding left the sum short of the goal: the last one there is)
  }
  __syncthreads();
  if (i < N) {
    // path: node 0 and the accepted nodes; tokens: theirs, then the last one
    p.path[(int64_t)b * N + i] = i >= count ? -1 : i == 0 ? 0 : path[i];
    const int64_t out = i + 1 < count ? (int64_t)tok[path[i + 1]] : i + 1 == count ? last : -1;
    token_store(p.tokens, p.token_bytes, (int64_t)b * N + i, out);
  }
  if (i == 0) p.counts[b] = count;
}

// Greedy: a child is accepted iff its token is the target's largest logit at
// its parent (the lowest index of equal ones; a NaN counts as largest).
__device__ __forceinline__ uint32_t logit_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (x == 0.f) return 0x80000000u;  // -0 and +0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// An entry as one comparable number: its key, then the complement of its index.
__device__ __forceinline__ uint64_t logit_entry(float x, int y) { return (uint64_t)logit_key(x) << 32 | (uint32_t)~y; }
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t wave_largest(uint64_t top) {
#pragma unroll
  for (int o = 32; o; o >>= 1) top = larger(top, (uint64_t)__shfl_xor((unsigned long long)top, o));
  return top;
}

// The largest entry of [lo, hi) of a row, hi > lo, among threads i, i + n, .. of
// n. A lane keeps its largest value (NaN wins, the first one) and the 16 bytes
// it stood in, two instructions an entry, and looks for the place in them at the
// end. Addresses past the last 16 bytes are moved back to them: what is seen
// twice changes nothing.
template <int DT>
__device__ __forceinline__ uint64_t largest_of(const typename ProbElt<DT>::T* P, int lo, int hi, int i, int n) {
  using E = ProbElt<DT>;
  constexpr int U = 8;
  if (hi - lo < E::V) return lo + i < hi ? logit_entry(E::at(P + lo + i), lo + i) : 0;
  float top = -__builtin_inff();
  int where = min(lo + i * E::V, hi - E::V);
  for (int at = lo; at < hi; at += n * E::V * U) {
    u32x4 a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = E::load(P + min(at + (n * u + i) * E::V, hi - E::V));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float m = E::get(a[u], 0);
#pragma unroll
      for (int e = 1; e < E::V; ++e) m = __builtin_elementwise_maximum(m, E::get(a[u], e));
      const bool more = top == top && !(m <= top);
      top = more ? m : top;
      where = more ? min(at + (n * u + i) * E::V, hi - E::V) : where;
    }
  }
  const u32x4 a = E::load(P + where);
  int y = 0;
#pragma unroll
  for (int e = E::V - 1; e >= 0; --e) {
    const float x = E::get(a, e);
    if (x == top || (x != x && top != top)) y = where + e;
  }
  return logit_entry(top, y);
}

// The largest entry of every part of every row of every tree, a wave each. Bound
// by the bytes of the logits: 53 MB in 11.7-12.4 us, 4.3 TB/s.
constexpr int kTopParts = 16;
template <int DT>
__global__ __launch_bounds__(256) void verify_tops_kernel(const VerifyParams p) {
  using T = typename ProbElt<DT>::T;
  constexpr int E = 64 * ProbElt<DT>::V;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = (int)(unit % kTopParts);
  const int64_t row = unit / kTopParts;
  const int b = (int)(row / p.N), node = (int)(row - (int64_t)b * p.N);  // (16 units a row: no workgroup hangs over)
  int own, unused;
  tree_node(p, b, node, own, unused);
  if (own < -1) return;  // no walk gets there
  const int per = ((p.V + kTopParts - 1) / kTopParts + E - 1) / E * E;
  const int lo = min(s * per, p.V), hi = min(lo + per, p.V);
  const T* const P = static_cast<const T*>(p.target) + (int64_t)b * p.ts0 + (int64_t)node * p.ts1;
  const uint64_t top = lo < hi ? wave_largest(largest_of<DT>(P, lo, hi, lane, 64)) : 0;
  if (lane == 0) p.tops[unit] = top;
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_greedy_kernel(const VerifyParams p) {
  using T = typename ProbElt<DT>::T;
  __shared__ int32_t par[kTreeMaxNodes], tok[kTreeMaxNodes], path[kTreeMaxNodes], best[kTreeMaxNodes];
  __shared__ uint64_t tops[2][kVerifyWaves];
  const int b = blockIdx.x, i = threadIdx.x, lane = i & 63;
  const int w = __builtin_amdgcn_readfirstlane(i >> 6);
  const int N = p.N;
  const T* const target = static_cast<const T*>(p.target) + (int64_t)b * p.ts0;
  if (i < N) tree_node(p, b, i, par[i], tok[i]);
  if (p.tops && i < N) {
    uint64_t top = 0;
#pragma unroll
    for (int x = 0; x < kTopParts; ++x) top = larger(top, p.tops[((int64_t)b * N + i) * kTopParts + x]);
    best[i] = (int)~(uint32_t)top;
  }
  __syncthreads();
  const bool active = par[0] == -1;
  int cur = 0, count = active ? 1 : 0, buf = 0;
  int64_t last = -1;
  while (active) {
    int t;
    if (p.tops) {
      t = best[cur];
    } else {
      uint64_t top = wave_largest(largest_of<DT>(target + (int64_t)cur * p.ts1, 0, p.V, i, kVerifyThreads));
      if (lane == 0) tops[buf][w] = top;
      __syncthreads();
      for (int x = 0; x < kVerifyWaves; ++x) top = larger(top, tops[buf][x]);
      buf ^= 1;  // (the next node's do not overwrite what another wave still reads)
      t = (int)~(uint32_t)top;
    }
    const int ch = next_child(par, N, cur, cur, lane, tok, t);
    if (ch < 0) {
      last = t;
      break;
    }
    cur = ch;
    if (i == 0) path[count] = cur;
    ++count;
  }
  __syncthreads();
  if (i < N) {
    p.path[(int64_t)b * N + i] = i >= count ? -1 : i == 0 ? 0 : path[i];
    const int64_t out = i + 1 < count ? (int64_t)tok[path[i + 1]] : i + 1 == count ? last : -1;
    token_store(p.tokens, p.token_bytes, (int64_t)b * N + i, out);
  }
  if (i == 0) p.counts[b] = count;
}

// All rows first or one after another on the walk? The first costs the bytes of
// the logits at 4.3 TB/s and a launch, whatever is accepted; the second 3 to 5 us
// a visited node of 128000 tokens, whose row one CU reads at some 80 GB/s, for the
// sequence that accepts most. All rows first while they are 64 MiB at most. Measured,
// bf16 (us, rows first / on the walk, 2 to 5 nodes visited): 128000 tokens, 1 x 26
// 12.9 / 25.2, 8 x 26 (53 MB) 16.9 / 26.7, 16 x 26 (106 MB) 26.5 / 25.6-28.2, 32 x 26
// 46.0 / 28.8; 32000 tokens, 1 x 8 12.5 / 13.2, 64 x 8 (33 MB) 13.9 / 16.3,
// 64 x 26 (106 MB) 26.9 / 20.2. Where the two meet depends on the nodes visited, which
// the host does not know: at 106 MB of the larger vocabulary they are equal, and a
// batch of few, deep paths would gain from rows first there.
size_t verify_tops_bytes(int B, int N, int V, int dtype) {
  const int64_t rows = (int64_t)B * N;
  if (rows > (64ll << 20) / ((int64_t)V * (dtype == 2 ? 4 : 2)) || rows > 1 << 20) return 0;  // (and one launch)
  return (size_t)rows * kTopParts * sizeof(uint64_t);
}

template <int DT>
static void launch_verify_t(const VerifyParams& p, int mode, hipStream_t stream) {
  const dim3 grid((unsigned)p.B), block(kVerifyThreads);
  if (mode == kDraftPicks) hipLaunchKernelGGL((verify_draft_kernel<DT, kDraftPicks>), grid, block, 0, stream, p);
  else if (mode == kDraftIid) hipLaunchKernelGGL((verify_draft_kernel<DT, kDraftIid>), grid, block, 0, stream, p);
  else if (mode == kDraftTree) hipLaunchKernelGGL((verify_draft_kernel<DT, kDraftTree>), grid, block, 0, stream, p);
  else {
    if (p.tops)
      hipLaunchKernelGGL((verify_tops_kernel<DT>), dim3((unsigned)((int64_t)p.B * p.N * kTopParts / 4)), dim3(256), 0,
                         stream, p);
    hipLaunchKernelGGL((verify_greedy_kernel<DT>), grid, block, 0, stream, p);
  }
}

hipError_t launch_verify(const VerifyParams& p, int mode, int dtype, hipStream_t stream) {
  if (dtype == 0) launch_verify_t<0>(p, mode, stream);
  else if (dtype == 1) launch_verify_t<1>(p, mode, stream);
  else launch_verify_t<2>(p, mode, stream);
  return hipGetLastError();
}

// ---- keeping the accepted path -------------------------------------------------
//
// Row base + path[j] of every layer's pools moves to row base + j, j < count.
// One thread owns one 16-byte column of one pool and walks j upward, so no
// other thread touches what it reads or writes; path[j] >= j and rising means
// that a row is read before an earlier place of it is overwritten: with eight
// rows in flight, rows j .. j + 7 are read before any of their places is
// written, and later ones come from rows behind all of those. The slots are
// looked up once per workgroup. Bound: bytes, where a batch moves many (32 trees in
// 32 layers, 33 MB, 8.5-9 us); three dependent reads (path, block id, row) otherwise
// (2.0-2.3 us).
constexpr int kKeepFlight = 8;

__global__ __launch_bounds__(256) void kv_keep_kernel(const KeepParams p) {
  __shared__ int64_t from[2][kTreeMaxNodes], to[2][kTreeMaxNodes];  // byte offsets in a K and a V pool, -1: stays
  __shared__ int steps;
  const int b = blockIdx.y;
  const int count = min(p.counts[b], p.N);
  if (threadIdx.x == 0) steps = 0;
  __syncthreads();
  const int start = p.starts[b];
  const int64_t limit = (int64_t)p.max_blocks * p.block_size;
  for (int j = threadIdx.x; j < count; j += 256) {
    const int node = p.path[(int64_t)b * p.ps0 + j];
    int64_t f[2] = {-1, -1}, t[2] = {-1, -1};
    const int64_t src = (int64_t)start + node, dst = (int64_t)start + j;
    if (start >= 0 && node > j && node < p.N && src < limit) {
      const int sb = (int)fdiv((uint32_t)src, p.bsdiv), db = (int)fdiv((uint32_t)dst, p.bsdiv);
      const int sid = p.bt[(int64_t)b * p.max_blocks + sb], did = p.bt[(int64_t)b * p.max_blocks + db];
      if ((uint32_t)sid < (uint32_t)p.num_blocks && (uint32_t)did < (uint32_t)p.num_blocks) {
        const int64_t so = src - (int64_t)sb * p.block_size, dofs = dst - (int64_t)db * p.block_size;
        for (int x = 0; x < 2; ++x) {
          f[x] = sid * p.block[x] + so * p.token[x];
          t[x] = did * p.block[x] + dofs * p.token[x];
        }
        atomicMax(&steps, j + 1);
      }
    }
    for (int x = 0; x < 2; ++x) from[x][j] = f[x], to[x][j] = t[x];
  }
  __syncthreads();
  const int n = steps;
  const uint32_t item = blockIdx.x * 256u + threadIdx.x;  // (layer, tensor, column)
  const uint32_t pool = fdiv(item, p.cprdiv), col = item - pool * p.cpr;
  if (pool >= 2u * (uint32_t)p.layers) return;
  const int x = (int)(pool & 1u);
  const uint32_t h = fdiv(col, p.cphdiv);
  char* const base = p.pools[pool] + (int64_t)h * p.head[x] + 16 * (int64_t)(col - h * p.cph);
  for (int j0 = 0; j0 < n; j0 += kKeepFlight) {
    u32x4 v[kKeepFlight];
#pragma unroll
    for (int u = 0; u < kKeepFlight; ++u)
      if (j0 + u < n && from[x][j0 + u] >= 0) v[u] = *reinterpret_cast<const u32x4*>(base + from[x][j0 + u]);
#pragma unroll
    for (int u = 0; u < kKeepFlight; ++u)
      if (j0 + u < n && from[x][j0 + u] >= 0) *reinterpret_cast<u32x4*>(base + to[x][j0 + u]) = v[u];
  }
}

hipError_t launch_kv_keep(const KeepParams& p, int B, hipStream_t stream) {
  const uint32_t items = 2u * (uint32_t)p.layers * p.cpr;
  hipLaunchKernelGGL(kv_keep_kernel, dim3((items + 255) / 256, (unsigned)B), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace cie
