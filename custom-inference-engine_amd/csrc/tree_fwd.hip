// Attention of a tree of drafted tokens over the paged KV cache, for gfx950.
//
// Every sequence has a history of base = ctx - N tokens and N nodes behind it,
// node i at position base + i of the pool. Query row (head h, node i) sees the
// history and the nodes whose bit is set in row i of the tree mask:
//   o = sum_j p_j v_j,  p = softmax over those j of q . k_j * scale.
// A row without a set bit is a padding slot of the batch: it sees nothing and
// its output is zero.
//
// Rows. The R = (Hq / Hk) * N query rows of a kv head are packed, r = g * N + i
// (query head kvh * group + g), so that every K / V byte a workgroup stages
// serves all of them. A wave holds 32 rows (one row per lane pair, see
// common.hpp), QT waves side by side cover a row tile of 32 QT rows of one kv
// head, and a workgroup takes HG kv heads: HG * QT waves. Rows beyond one tile
// go to workgroups of their own.
//
// Keys. A piece, one workgroup's work, is a run of 32-token tiles of ONE
// sequence. Every workgroup finds its own from the context lengths: with C tiles
// per piece, sequence b has ceil(tiles_b / C) pieces of nearly equal length, so
// ragged batches balance and the host needs no lengths. The launch has workgroups
// for B + extra pieces, enough for C = ceil(all tiles / extra) whatever the lengths.
// (The smallest C that they are enough for, found by bisection, takes a tenth off
// the longest piece and nothing off the time: the whole chip's rate bounds it.) A
// sequence of more pieces than one leaves partial states (acc, m, l) that
// tree_merge_kernel combines in a fixed order.
//
// Per tile: K and V go global -> LDS by 16-byte direct copies into a ring of NST
// stages,
//   S^T = K Q^T, online softmax in registers, O^T += V^T P^T
// as in paged_fwd.hip. Only tiles that reach past the history look at the tree
// mask: the 32 bits of every row and tile are cut out of its words before the loop.
//
// Bounds. Few rows per kv head: the K / V bytes (32 trees of 16 nodes over 256-4096
// tokens, 32/8 heads, D = 64: 141 MB, main pass 37-38 us, 3.8 TB/s). Many rows: products
// and softmax, which overlap in part only (four trees of 64 nodes over 8192-16384 tokens,
// 32/8 heads, D = 128: 55 GFLOP, half as much again with the second part of P; main pass
// 91-100 us, the first tile arriving after 6.5, the partial states 33 MB). Short ones:
// the start, four dependent reads (lengths, block ids, first tile, then the partial
// states of the merge).
//
// P keeps two 16-bit parts for the second product, the rounded p and what the
// rounding left (Elt::rest2), with a product for each; its sum is fp32 and of the
// unrounded values. The output is then within its own rounding of the fp32 formula.
// Relative error against 64 bits, one part / two parts / the output's rounding alone:
// 32 x 16 in fp16 2.90e-4 / 2.07e-4 / 2.07e-4, 4 x 64 in bf16 2.34e-3 / 1.66e-3 /
// 1.66e-3; time of the two calls 39.4 / 42.1 and 81.7 / 99.0 us. A seen V that is not
// finite leaves its column of the row not finite: an infinity may come out as NaN,
// its products with the two parts being of either sign.
//
// A masked key must not reach a row even if its V holds infinities or NaN (the
// slots of padding nodes are never written): in a tile past the history such
// values are taken out in LDS before the product and added at the end for the rows
// that see their key.
#include <climits>
#include <type_traits>

#include "kernels.hpp"
#include "rope.hpp"

namespace cie {

constexpr float kLazyRescaleTree = 8.0f;  // log2: the running maximum is replaced only when it is this much behind

template <int D, int QT>
struct TreeCfg {
  static constexpr int KK = D / 16;                // MFMA steps over head_dim
  static constexpr int DT = D >= 32 ? D / 32 : 1;  // 32-column output tiles
  static constexpr int S = D / 8;                  // 16-byte chunks per head row
  static constexpr int QTI = QT < D / 16 ? QT : D / 16;  // waves of a head that issue its copies
  static constexpr bool PAIR = QT == 8;            // two waves a SIMD, half a step apart
  static constexpr int CPW = D / (16 * QTI);             // 1 KiB copies per issuing wave, tensor and tile
};

__device__ __forceinline__ bool tree_ctx_valid(const TreeParams& p, int ctx) {
  return ctx >= p.N && ctx <= p.ctx_limit && p.num_blocks > 0;
}

// The 32 mask bits of keys rel0 .. rel0 + 31 (node indices; the history's are
// negative and visible) for the row whose words start at `words`.
__device__ __forceinline__ uint32_t tree_bits(const int32_t* words, int rel0, int N, int W, bool node_row) {
  if (!node_row) return 0u;
  const int lo = rel0 < 0 ? 0 : rel0;
  const int w0 = lo >> 5, sh = lo & 31;
  const uint32_t a = w0 < W ? (uint32_t)words[w0] : 0u;
  const uint32_t b = w0 + 1 < W ? (uint32_t)words[w0 + 1] : 0u;
  uint32_t x = sh ? (a >> sh) | (b << (32 - sh)) : a;  // nodes lo ..
  const int left = N - lo;                             // nodes at and after lo
  if (left < 32) x &= left > 0 ? (1u << left) - 1u : 0u;
  if (rel0 < 0) x = rel0 > -32 ? (x << -rel0) | ((1u << -rel0) - 1u) : 0xffffffffu;
  return x;
}

// 16-bit values with all exponent bits set are infinities and NaN.
template <int DTYPE>
constexpr uint32_t kExp = DTYPE == 0 ? 0x7c00u : 0x7f80u;
template <int DTYPE>
__device__ __forceinline__ bool all_finite(u32x4 v) {
  bool ok = true;
#pragma unroll
  for (int y = 0; y < 4; ++y)
    ok &= (v[y] & kExp<DTYPE>) != kExp<DTYPE> && (v[y] >> 16 & kExp<DTYPE>) != kExp<DTYPE>;
  return ok;
}
template <int DTYPE>
__device__ __forceinline__ u32x4 finite_or_zero(u32x4 v) {
#pragma unroll
  for (int y = 0; y < 4; ++y)
    v[y] = ((v[y] & kExp<DTYPE>) != kExp<DTYPE> ? v[y] & 0xffffu : 0u) |
           ((v[y] >> 16 & kExp<DTYPE>) != kExp<DTYPE> ? v[y] & 0xffff0000u : 0u);
  return v;
}
template <int DTYPE>
__device__ __forceinline__ float widen(uint32_t h) {
  return DTYPE == 0 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
}

// Whether row i's mask has a bit among the N nodes.
__device__ __forceinline__ bool tree_row_live(const int32_t* words, int N) {
  uint32_t any = 0;
  for (int w = 0; w < (N >> 5); ++w) any |= (uint32_t)words[w];
  if (N & 31) any |= (uint32_t)words[N >> 5] & ((1u << (N & 31)) - 1u);
  return any != 0;
}

// Rotary position of a node; a sum past 31 bits is past every table.
__device__ __forceinline__ int tree_position(int base, int depth) {
  return (int)min((uint32_t)base + (uint32_t)max(depth, 0), 0x7fffffffu);
}

// Waits for a tile, `ahead` tiles having been issued after it, of PT copies each
// (vmcnt counts them). It leaves three of those outstanding at most: with a ring of
// more than six stages (seven for QT = 8) a step also waits for tiles that it does not
// need yet, and at D = 256 with QT = 1, whose PT is 32, the first wait is for all tiles
// issued.
template <int PT>
__device__ __forceinline__ void tree_wait(int ahead) {
  if constexpr (3 * PT < 64) {
    if (ahead >= 3) { vm_wait<3 * PT>(); return; }
  }
  if constexpr (2 * PT < 64) {
    if (ahead == 2) { vm_wait<2 * PT>(); return; }
  }
  if (ahead == 1) { vm_wait<PT>(); return; }
  vm_wait<0>();
}

// Writes 16-bit pattern pairs into this lane's half of an output row.
template <int D>
__device__ __forceinline__ void tree_fill(uint16_t* row, int hl, uint32_t bits2) {
#pragma unroll
  for (int d = hl * (D / 2); d < (hl + 1) * (D / 2); d += 8)
    *reinterpret_cast<u32x4*>(row + d) = u32x4{bits2, bits2, bits2, bits2};
}

template <int DTYPE, int D, int QT>
__global__ __launch_bounds__(tree_threads(D, QT)) void tree_fwd_kernel(const TreeParams p) {
  warm_kernargs<sizeof(TreeParams)>();
  using C = TreeCfg<D, QT>;
  using E = Elt<DTYPE>;
  // the ring first (its stages then lie at multiples of their power-of-two size,
  // so that the swizzles below are an XOR of the address), the block ids behind it
  extern __shared__ __attribute__((aligned(1024))) uint16_t ring[];
  int32_t* const sbt = reinterpret_cast<int32_t*>(ring + p.NST * (2 * kPagedTile * 8) * p.NCH);
  uint32_t* const odd = reinterpret_cast<uint32_t*>(sbt + kTreeIds);  // [HG][kTreeOddWords] keys whose V is not finite
  uint32_t* const seen = odd + p.HG * kTreeOddWords;                  // [tile past the history][32 QT rows] mask bits

  // (piece j, head group gh) = unit u, row tile rt; the row tiles of a unit are
  // 2^xcd_shift workgroup ids apart, so that they share an XCD's L2
  const int nx = 1 << p.xcd_shift;
  int u = blockIdx.x, rt = 0;
  if (p.NRT > 1) {
    const int per = nx * p.NRT, grp = u / per, rem = u - grp * per;
    rt = rem >> p.xcd_shift;
    u = grp * nx + (rem & (nx - 1));
  }
  const int j = u / p.NG, gh = u - j * p.NG;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hl = lane >> 5;
  const int hh = w / QT, qt = w % QT;
  const int kvh = gh * p.HG + hh;
  const uint32_t nan2 = 0x7fff7fffu;  // NaN in both 16-bit types

  // ---- this workgroup's piece ------------------------------------------------
  int NT = 0, ctx0 = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    const int ctx = b < p.B ? p.lens[b] : -1;
    if (b0 == 0) ctx0 = ctx;
    const int incl = wave_incl_scan(tree_ctx_valid(p, ctx) ? (ctx + kPagedTile - 1) / kPagedTile : 0);
    NT += __builtin_amdgcn_readlane(incl, 63);
  }
  const int CT = max(p.cmin, (int)(((uint32_t)NT + (uint32_t)p.extra - 1) / (uint32_t)p.extra));
  int carry = 0, b = -1, ctx = 0, t = 0, n = 0, j0 = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int bb = b0 + lane;
    const int cx = b0 == 0 ? ctx0 : (bb < p.B ? p.lens[bb] : -1);
    const int tb = tree_ctx_valid(p, cx) ? (cx + kPagedTile - 1) / kPagedTile : 0;
    const int nb = bb < p.B ? max(1, (int)(((uint32_t)tb + (uint32_t)CT - 1) / (uint32_t)CT)) : 0;
    const int incl = wave_incl_scan(nb);
    const int pre = carry + incl - nb;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(nb > 0 && pre <= j && j < pre + nb);
    if (hit) {
      const int hlane = __builtin_ctzll(hit);
      b = b0 + hlane;
      ctx = __builtin_amdgcn_readlane(cx, hlane);
      t = __builtin_amdgcn_readlane(tb, hlane);
      n = __builtin_amdgcn_readlane(nb, hlane);
      j0 = __builtin_amdgcn_readlane(pre, hlane);
      break;
    }
    carry += __builtin_amdgcn_readlane(incl, 63);
  }
  if (b < 0) return;  // the launch has a workgroup for every piece there can be
  if (p.info && j == j0 && gh == 0 && rt == 0 && threadIdx.x == 0) p.info[b] = int2{j0, n};

  // ---- query row -------------------------------------------------------------
  const int r = (rt * QT + qt) * 32 + l32;
  const bool rv = r < p.R;
  const int g = rv ? (int)fdiv((uint32_t)r, p.ndiv) : 0;
  const int node = rv ? r - g * p.N : 0;
  const int hq = kvh * p.group + g;
  const int32_t* const words = p.mask + (int64_t)b * p.ms0 + (int64_t)node * p.ms1;
  auto out_row = [&] { return p.o + (int64_t)b * p.os0 + hq * p.os1 + (int64_t)node * p.os2; };
  const bool live = tree_row_live(words, p.N);
  if (t == 0) {  // an invalid context length
    if (rv) tree_fill<D>(out_row(), hl, live ? nan2 : 0u);
    return;
  }
  const int per_piece = (int)(((uint32_t)t + (uint32_t)n - 1) / (uint32_t)n);
  const int tlo = (j - j0) * per_piece, thi = min(t, tlo + per_piece), T = thi - tlo;
  const int base = ctx - p.N;

  // ---- block ids of the piece, query fragments ----------------------------------
  // What depends on the piece alone is asked for at once: block ids, q, depth. The
  // rotation's table entries follow, then the first copies; q is rotated behind them
  // (waiting for each in turn, the start took two more round trips to memory).
  const int blk_lo = (int)fdiv((uint32_t)(kPagedTile * tlo), p.bsdiv);
  const int nids = (int)fdiv((uint32_t)(min(ctx, kPagedTile * thi) - 1), p.bsdiv) - blk_lo + 1;
  const int32_t* const src = p.bt + (int64_t)b * p.max_blocks + blk_lo;
  const int id0 = src[min((int)threadIdx.x, nids - 1)];
  u32x4 qf[C::KK];
  const uint16_t* const qrow = p.q + (int64_t)b * p.qs0 + hq * p.qs1 + (int64_t)node * p.qs2;
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) qf[kk] = load16(qrow + 16 * kk + 8 * hl, rv);
  const int depth = p.rope.cos ? p.depths[(int64_t)b * p.ds0 + node] : 0;
  if ((int)threadIdx.x < nids) sbt[threadIdx.x] = (uint32_t)id0 < (uint32_t)p.num_blocks ? id0 : -1;
  for (int x = threadIdx.x + blockDim.x; x < nids; x += blockDim.x) {
    const int id = src[x];
    sbt[x] = (uint32_t)id < (uint32_t)p.num_blocks ? id : -1;
  }
  for (int x = threadIdx.x; x < p.HG * kTreeOddWords; x += blockDim.x) odd[x] = 0;
  const int whole = min(max(base / kPagedTile - tlo, 0), T);  // tiles of history alone
  // the mask bits of the other tiles, a row's once for all heads (read from memory in
  // the loop, they waited there for every copy under way)
  if (hh == 0 && hl == 0)
#pragma unroll 4
    for (int x = whole; x < T; ++x)
      seen[(x - whole) * (32 * QT) + 32 * qt + l32] = tree_bits(words, kPagedTile * (tlo + x) - base, p.N, p.W, live);
  RopeRow<D> rr;
  if (p.rope.cos) rr = rope_row_load<D>(p.rope, tree_position(base, depth), hl);
  __syncthreads();
  bool bad = false;
  for (int x = lane; x < nids; x += 64) bad |= sbt[x] < 0;
  const bool poison = __builtin_amdgcn_ballot_w64(bad) != 0;  // an id outside the pool: NaN rows, never a read

  // ---- copies ----------------------------------------------------------------
  const int NCH = p.NCH, NST = p.NST;
  const int lg_nch = __builtin_ctz(NCH);
  const int TILE_EL = kPagedTile * NCH * 8;
  const int STAGE_EL = 2 * TILE_EL;
  const bool issuer = qt < C::QTI;
  const int c0 = (hh * C::QTI + qt) * C::CPW;  // this wave's first copy of a tensor's tile
  // chunk P = 64 (c0 + x) + lane of the tile: token P / NCH, stored chunk P % NCH of
  // its row, which holds chunk (P % NCH) ^ row_swizzle(token); NCH divides 64
  const int tok0 = (64 * c0 + lane) >> lg_nch, tok_step = 64 >> lg_nch, chunk0 = lane & (NCH - 1);
  const uint16_t* const kbase = p.kc + (int64_t)gh * p.HG * p.ks2;
  const uint16_t* const vbase = p.vc + (int64_t)gh * p.HG * p.vs2;
  // Whole tiles of a pool that 32-bit byte offsets reach, K and V laid out alike,
  // blocks a multiple or a divisor of the tile: per copy one block id and one
  // multiply-add, everything else of the address is the lane's own (without this
  // the addresses took more of a step than its softmax).
  uint32_t lofs[C::CPW];
  int lblk[C::CPW];
#pragma unroll
  for (int x = 0; x < C::CPW; ++x) {
    const int tk = tok0 + x * tok_step;
    const int cx = chunk0 ^ row_swizzle(NCH, tk);
    lblk[x] = (int)fdiv((uint32_t)tk, p.bsdiv);
    lofs[x] = 2u * (uint32_t)((tk - lblk[x] * p.block_size) * (int)p.ks1 + (cx / C::S) * (int)p.ks2 + 8 * (cx % C::S));
  }
  const uint32_t ring_lds = lds_addr_of(ring);
  int i_stage = 0;
  auto issue = [&](int k) __attribute__((always_inline)) {
    const int tbase = kPagedTile * (tlo + k);
    const uint32_t st = ring_lds + 2u * (uint32_t)(i_stage * STAGE_EL) + 1024u * (uint32_t)c0;
    i_stage = i_stage + 1 == NST ? 0 : i_stage + 1;
    if (p.narrow && tbase + kPagedTile <= ctx) {
      const int blk = (int)fdiv((uint32_t)tbase, p.bsdiv);
      const uint32_t in = 2u * (uint32_t)((tbase - blk * p.block_size) * (int)p.ks1);  // 0 unless blocks are larger
      uint32_t off[C::CPW];
#pragma unroll
      for (int x = 0; x < C::CPW; ++x)
        off[x] = __umul24((uint32_t)max(sbt[blk - blk_lo + lblk[x]], 0), p.ks0_24) + lofs[x] + in;
#pragma unroll
      for (int x = 0; x < C::CPW; ++x) {
        dma16_sv_nt(kbase, off[x], st + 1024u * x);
        dma16_sv_nt(vbase, off[x], st + 2u * TILE_EL + 1024u * x);
      }
      return;
    }
    for (int x = 0; x < C::CPW; ++x) {
      const int tk = min(tbase + tok0 + x * tok_step, ctx - 1);
      const int blk = (int)fdiv((uint32_t)tk, p.bsdiv), off = tk - blk * p.block_size;
      const int bid = max(sbt[blk - blk_lo], 0);
      const int cx = chunk0 ^ row_swizzle(NCH, tok0 + x * tok_step);
      const int hd = cx / C::S, dc = 8 * (cx % C::S);
      dma16_at_nt(kbase + (int64_t)bid * p.ks0 + (int64_t)off * p.ks1 + hd * (int32_t)p.ks2 + dc, st + 1024u * x);
      dma16_at_nt(vbase + (int64_t)bid * p.vs0 + (int64_t)off * p.vs1 + hd * (int32_t)p.vs2 + dc,
                  st + 2u * TILE_EL + 1024u * x);
    }
  };
  const int reach = NST - (C::PAIR ? 2 : 1);  // step k copies tile k + reach
  if (issuer)
    for (int k = 0; k < min(reach, T); ++k) issue(k);
  if (p.rope.cos) rope_row_apply<DTYPE, D>(qf, p.rope, rr, rv, hl);
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) qf[kk] ^= u32x4{p.q_sign, p.q_sign, p.q_sign, p.q_sign};

  // ---- tile loop -------------------------------------------------------------
  // Byte addresses inside a tile. K row l32, chunk hh S + 2 kk + hl: the kk part is
  // an XOR of the address. V^T fragment (dt, cc): lane (group gq, row rq of it) points
  // at token 16 cc + 4 hl + rq / 4 (and 8 on), dims 32 dt + 16 (gq & 1) + 4 (rq % 4)
  // (the dt part an XOR too); the transpose read hands each lane four keys of dim
  // 32 dt + l32.
  const uint32_t k_lane = 16u * (uint32_t)((l32 << lg_nch) + ((hh * C::S + hl) ^ row_swizzle(NCH, l32)));
  uint32_t v_lane[2][2];
  {
    const int rq = lane & 15, gq = lane >> 4;
    int d = 16 * (gq & 1) + 4 * (rq & 3);
    if (D < 32) d = min(d, D - 4);  // rows >= D of O^T are discarded
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int up = 0; up < 2; ++up) {
        const int tk = 16 * cc + 4 * hl + (rq >> 2) + 8 * up;
        v_lane[cc][up] = 2u * (uint32_t)TILE_EL +
                         16u * (uint32_t)((tk << lg_nch) + ((hh * C::S + (d >> 3)) ^ row_swizzle(NCH, tk))) + 2u * (d & 7);
      }
  }
  f32x16 acc[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt) acc[dt] = f32x16{};
  float mx = -INFINITY, l = 0.f;
  const float c = p.scale_log2;
  f32x16 sc = f32x16{}, sn;      // scores of the tile, then its probabilities; scores of the next one
  u32x4 pb[2] = {}, pr[2] = {};  // the probabilities in 16 bits, and what that rounding left

  // V of a tile past the history, before any wave reads it: values that are not
  // finite become zeros in LDS and their keys are noted, this wave's share of the
  // tile's tokens.
  auto tidy = [&](int k, int st) __attribute__((always_inline)) {
    uint16_t* const vst = ring + st * STAGE_EL + TILE_EL;
    constexpr int TOK = kPagedTile / QT;
    for (int x = lane; x < TOK * C::S; x += 64) {
      const int tk = qt * TOK + x / C::S, cc = (hh * C::S + x % C::S) ^ row_swizzle(NCH, tk);
      u32x4* const at = reinterpret_cast<u32x4*>(vst + ((tk << lg_nch) + cc) * 8);
      const u32x4 v = *at;
      if (!all_finite<DTYPE>(v)) {
        *at = finite_or_zero<DTYPE>(v);
        atomicOr(&odd[hh * kTreeOddWords + (k - whole)], 1u << tk);
      }
    }
  };
  // Step k: the matrix part, scores of tile k and values of tile k - 1, then the
  // softmax of tile k. Fragments are read from LDS ahead of their products: V of tile
  // k - 1 between the products of the scores, K of tile k + 1 between the pieces of
  // the softmax (read right before use, the LDS latency stood in front of every
  // product; read all at once, the LDS bandwidth in front of the rest).
  //
  // One barrier a step, between the two parts: behind it every wave has read V of tile
  // k - 1 (whose stage the softmax part refills) and every wave's copies of tile k + 1
  // are done. With two waves on a SIMD (QT = 8) the second one takes its matrix part
  // behind the barrier, so that it multiplies while the first one is in its softmax;
  // the ring then refills a stage one step later. The matrix part runs at a raised
  // wave priority: the products are issued first, the other wave's softmax in between.
  // Four trees of 64 nodes over 8192-16384 tokens, with P in one part: 86 us in step, 84.5 half a step
  // apart, 81.5 with the priority. (Two halves kept apart by a barrier after each part:
  // 90; they wait for one another more than they overlap.)
  u32x4 vf[2 * C::DT], kf[C::KK];
  auto load_key = [&](int st, int kk) __attribute__((always_inline)) {
    kf[kk] = lds_read16_at((ring_lds + 2u * (uint32_t)(st * STAGE_EL) + k_lane) ^ (32u * kk));
  };
  auto load_value = [&](int st, int f) __attribute__((always_inline)) {
    const uint32_t sp = ring_lds + 2u * (uint32_t)(st * STAGE_EL);
    const u32x2 lo = lds_read_tr16_at((sp + v_lane[f & 1][0]) ^ (64u * (f >> 1)));
    const u32x2 hi = lds_read_tr16_at((sp + v_lane[f & 1][1]) ^ (64u * (f >> 1)));
    vf[f] = u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  if (issuer) tree_wait<2 * C::CPW>(min(reach - 1, T - 1));
  __syncthreads();
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk) load_key(0, kk);
  if (whole == 0) tidy(0, 0);
  int st_cur = 0, st_prev = 0;  // stages of tiles k and k - 1
  auto values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) acc[dt] = E::mfma(vf[2 * dt + cc], pb[cc], acc[dt]);
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) acc[dt] = E::mfma(vf[2 * dt + cc], pr[cc], acc[dt]);
  };
  // What the rounding of probabilities 2 w2 and 2 w2 + 1 left. A wave that has its SIMD
  // to itself takes it between the score products of the next tile, which do not need
  // the vector unit; two that share one in the softmax part, where the other wave
  // multiplies (48 trees of 8 nodes over 4000 tokens, 32/8 heads, D = 128, all in the
  // softmax part 148 -> 142 us; 4 x 64, all between the products 99 -> 103).
  auto rest = [&](int w2) __attribute__((always_inline)) {
    pr[w2 >> 2][w2 & 3] = E::rest2(pb[w2 >> 2][w2 & 3], sc[2 * w2], sc[2 * w2 + 1]);
  };
  auto matrix = [&](int k) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
    sn = f32x16{};
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      sn = E::mfma(kf[kk], qf[kk], sn);
      if (kk < 2 * C::DT) load_value(st_prev, kk);
      if (!C::PAIR)
#pragma unroll
        for (int w2 = 8 * kk / C::KK; w2 < 8 * (kk + 1) / C::KK; ++w2) rest(w2);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (D < 32) load_value(st_prev, 1);
    if (k > 0) values();
    sc = sn;
    __builtin_amdgcn_s_setprio(0);
  };
  const bool late = C::PAIR && w >= 4;
  for (int k = 0; k < T; ++k) {
    if (!late) matrix(k);
    const int st_next = st_cur + 1 == NST ? 0 : st_cur + 1;
    if (issuer && k + 1 < T) tree_wait<2 * C::CPW>(min(reach - 2, T - 2 - k));
    __syncthreads();
    if (issuer && k + reach < T) issue(k + reach);
    if (k + 1 >= whole && k + 1 < T) tidy(k + 1, st_next);
    if (late) matrix(k);
    if (k >= whole) {  // the tile reaches past the history: the row's mask decides
      const uint32_t vis = seen[(k - whole) * (32 * QT) + 32 * qt + l32] >> (4 * hl);
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = (vis >> (8 * (e >> 2) + (e & 3))) & 1u ? sc[e] : -INFINITY;
    }
    const float mxs = xhalf_max(max16(sc)) * c;
    const bool grow = mxs > mx + kLazyRescaleTree;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float m_new = grow ? mxs : mx;
      const float alpha = grow ? exp2_fast(mx - m_new) : 1.f;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) acc[dt] *= alpha;
      mx = m_new;
    }
    const float neg_m = mx == -INFINITY ? 0.f : -mx;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
#pragma unroll
      for (int kk = 0; kk < C::KK; ++kk)
        if (kk * 4 / (C::KK < 4 ? 4 : C::KK) == e4) load_key(st_next, kk);  // (of the last tile: of no use)
#pragma unroll
      for (int e = 4 * e4; e < 4 * e4 + 4; ++e) sc[e] = exp2_fast(fmaf(sc[e], c, neg_m));
      l += (sc[4 * e4] + sc[4 * e4 + 1]) + (sc[4 * e4 + 2] + sc[4 * e4 + 3]);
#pragma unroll
      for (int w2 = 2 * e4; w2 < 2 * e4 + 2; ++w2) {
        pb[w2 >> 2][w2 & 3] = E::pack2(sc[2 * w2], sc[2 * w2 + 1]);
        if (C::PAIR) rest(w2);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    st_prev = st_cur;
    st_cur = st_next;
  }
#pragma unroll
  for (int f = 0; f < 2 * C::DT; ++f) load_value(st_prev, f);
  if (!C::PAIR)
#pragma unroll
    for (int w2 = 0; w2 < 8; ++w2) rest(w2);
  values();

  // ---- values that are not finite ----------------------------------------------
  if (whole < T) {
    __syncthreads();
    for (int x = 0; x < T - whole; ++x)
      for (uint32_t keys = odd[hh * kTreeOddWords + x]; keys; keys &= keys - 1) {
        // the row's probability of that key once more, for the columns taken out
        const int key = kPagedTile * (tlo + whole + x) + __builtin_ctz(keys), a = key - base;
        if (key >= ctx) continue;  // (a copy of the last token)
        const int blk = (int)fdiv((uint32_t)key, p.bsdiv), off = key - blk * p.block_size;
        const int64_t id = max(sbt[blk - blk_lo], 0);
        const uint16_t* krow = p.kc + id * p.ks0 + (int64_t)off * p.ks1 + (int64_t)kvh * p.ks2;
        const uint16_t* vrow = p.vc + id * p.vs0 + (int64_t)off * p.vs1 + (int64_t)kvh * p.vs2;
        float s = 0.f;
#pragma unroll
        for (int kk = 0; kk < C::KK; ++kk) {
          const f32x8 kv = widen8<DTYPE>(load16_clamped(krow + 16 * kk + 8 * hl)), qv = widen8<DTYPE>(qf[kk]);
#pragma unroll
          for (int y = 0; y < 8; ++y) s = fmaf(kv[y], qv[y], s);
        }
        s = xhalf_sum(s) * c;
        const bool sees = live && (a < 0 || (words[a >> 5] >> (a & 31)) & 1);
        const float pe = exp2_fast(s - (mx == -INFINITY ? 0.f : mx));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
          for (int g4 = 0; g4 < 4; ++g4) {
            const int d = 32 * dt + 8 * g4 + 4 * hl;
            const u32x2 v4 = *reinterpret_cast<const u32x2*>(vrow + min(d, D - 4));
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t h = y & 1 ? v4[y >> 1] >> 16 : v4[y >> 1] & 0xffffu;
              const float add = pe * widen<DTYPE>(h);
              acc[dt][4 * g4 + y] += (sees & ((h & kExp<DTYPE>) == kExp<DTYPE>)) ? add : 0.f;
            }
          }
      }
  }

  // ---- output ----------------------------------------------------------------
  const float lt = xhalf_sum(l);
  if (!rv) return;
  if (n == 1) {
    uint16_t* const orow = out_row();
    if (!live) {
      tree_fill<D>(orow, hl, 0u);
      return;
    }
    const float inv = poison ? __builtin_nanf("") : 1.f / lt;
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const int d = 32 * dt + 8 * g4 + 4 * hl;
        if (D >= 32 || d < D)
          *reinterpret_cast<u32x2*>(orow + d) =
              u32x2{E::pack2(acc[dt][4 * g4] * inv, acc[dt][4 * g4 + 1] * inv),
                    E::pack2(acc[dt][4 * g4 + 2] * inv, acc[dt][4 * g4 + 3] * inv)};
      }
    return;
  }
  // a partial state in lane order, 1 KiB a store: [row group][column group][lane][4]
  const int64_t slot = ((int64_t)j * p.Hk + kvh) * p.G32 + (rt * QT + qt);
  float* const part = p.part + slot * (32 * D) + 4 * lane;
  const float pz = poison ? __builtin_nanf("") : 1.f;
#pragma unroll
  for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      if (D >= 32 || g4 < D / 8)
        *reinterpret_cast<float4*>(part + 256 * (4 * dt + g4)) =
            float4{acc[dt][4 * g4] * pz, acc[dt][4 * g4 + 1] * pz, acc[dt][4 * g4 + 2] * pz, acc[dt][4 * g4 + 3] * pz};
  if (hl == 0) p.ml[slot * 32 + l32] = float2{mx * pz, lt * pz};
}

// Writes the nodes' K and V behind the history before attention reads them:
// node i of sequence b (rows b * N + i of kn / vn) to position base + i, K
// rotated at base + its depth. One thread moves a pair of 16-byte chunks (the
// two halves that a rotation mixes) of K and of V. Bound by latency: 2.4 us for 1 x 8
// nodes of 8 x 64, 3.4-4.9 for 8 x 26 of 8 x 128. Padding slots, positions
// outside the rotary tables and invalid sequences are left as they are.
template <int DTYPE>
__global__ __launch_bounds__(256) void tree_append_kernel(const TreeParams p) {
  warm_kernargs<sizeof(TreeParams)>();
  const int b = blockIdx.y;
  const uint32_t x = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = fdiv(x, p.updiv);  // node
  if (row >= (uint32_t)p.N) return;
  // (everything that depends on the arguments alone is asked for before anything is
  // waited for; block id and table entries, which depend on the length, together)
  const int ctx = p.lens[b];
  const int depth = p.rope.cos ? p.depths[(int64_t)b * p.ds0 + row] : 0;
  const uint32_t c = x - row * p.updiv.d;
  const int half = p.D / 2, h = (int)(c / (uint32_t)(p.D / 16)), d = 8 * (int)(c % (uint32_t)(p.D / 16));
  const int64_t r = (int64_t)b * p.N + row;
  const uint16_t* ks = p.kn + r * p.kns0 + h * p.kns1 + d;
  const uint16_t* vs = p.vn + r * p.vns0 + h * p.vns1 + d;
  u32x4 k0 = *reinterpret_cast<const u32x4*>(ks), k1 = *reinterpret_cast<const u32x4*>(ks + half);
  const u32x4 v0 = *reinterpret_cast<const u32x4*>(vs), v1 = *reinterpret_cast<const u32x4*>(vs + half);
  const bool live = tree_row_live(p.mask + (int64_t)b * p.ms0 + (int64_t)row * p.ms1, p.N);
  if (!tree_ctx_valid(p, ctx) || !live) return;
  const int pos = ctx - p.N + (int)row;
  const int blk = (int)fdiv((uint32_t)pos, p.bsdiv), off = pos - blk * p.block_size;
  const int id = p.bt[(int64_t)b * p.max_blocks + blk];
  if (p.rope.cos) {
    const int at = tree_position(ctx - p.N, depth);
    if (at >= p.rope.rows) return;
    rope_apply8<DTYPE>(k0, k1, rope_load(p.rope, (int64_t)at * half + d), p.rope.dt);
  }
  if ((uint32_t)id >= (uint32_t)p.num_blocks) return;
  uint16_t* kd = const_cast<uint16_t*>(p.kc) + (int64_t)id * p.ks0 + (int64_t)off * p.ks1 + (int64_t)h * p.ks2 + d;
  uint16_t* vd = const_cast<uint16_t*>(p.vc) + (int64_t)id * p.vs0 + (int64_t)off * p.vs1 + (int64_t)h * p.vs2 + d;
  *reinterpret_cast<u32x4*>(kd) = k0;
  *reinterpret_cast<u32x4*>(kd + half) = k1;
  *reinterpret_cast<u32x4*>(vd) = v0;
  *reinterpret_cast<u32x4*>(vd + half) = v1;
}

// Combines the pieces of every sequence that has more than one: a workgroup
// takes one column group (8 columns of 32 rows, 64 lanes x 4 values) and its
// four waves the pieces in turn, each reading whole 1 KiB runs of the partial
// states; the four results are joined in wave order. A launch and two dependent
// reads (2.4-3.3 us), then the bytes: 33 MB in 9.2-9.7 us. (One wave a group, a quarter
// of the workgroups: 10.0 -> 9.8 us there, 4.0 -> 4.7 at 13 pieces of 8 rows.)
constexpr int kTreeMergeWaves = 4, kTreeMergeBatch = 4;

template <int DTYPE, int D>
__global__ __launch_bounds__(64 * kTreeMergeWaves) void tree_merge_kernel(const TreeParams p) {
  using E = Elt<DTYPE>;
  __shared__ float4 sa[kTreeMergeWaves][64];
  __shared__ float2 sm[kTreeMergeWaves][64];
  const int b = blockIdx.y;
  const int2 inf = p.info[b];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hl = lane >> 5;
  const int cg = blockIdx.x % (D / 8), rg = blockIdx.x / (D / 8);  // rg = kvh * G32 + row group
  const int kvh = rg / p.G32, r = (rg - kvh * p.G32) * 32 + l32;
  const int g = (int)fdiv((uint32_t)r, p.ndiv), i = r - g * p.N;
  // (asked for along with the piece count, not after the last partial state)
  const bool live = w == 0 && r < p.R && tree_row_live(p.mask + (int64_t)b * p.ms0 + (int64_t)i * p.ms1, p.N);
  if (inf.y < 2) return;  // written whole by the main pass
  float M = -INFINITY, L = 0.f;
  float4 A = {0.f, 0.f, 0.f, 0.f};
  if (r < p.R)
    for (int k0 = w; k0 < inf.y; k0 += kTreeMergeWaves * kTreeMergeBatch) {
      float2 ml[kTreeMergeBatch];
      float4 a[kTreeMergeBatch];
#pragma unroll
      for (int u = 0; u < kTreeMergeBatch; ++u)
        if (k0 + kTreeMergeWaves * u < inf.y) {
          const int64_t slot = (int64_t)(inf.x + k0 + kTreeMergeWaves * u) * p.Hk * p.G32 + rg;
          ml[u] = p.ml[slot * 32 + l32];
          a[u] = *reinterpret_cast<const float4*>(p.part + slot * (32 * D) + 256 * cg + 4 * lane);
        }
#pragma unroll
      for (int u = 0; u < kTreeMergeBatch; ++u)
        if (k0 + kTreeMergeWaves * u < inf.y) merge_state(M, L, A, ml[u].x, ml[u].y, a[u]);
    }
  sa[w][lane] = A;
  sm[w][lane] = float2{M, L};
  __syncthreads();
  if (w != 0 || r >= p.R) return;
#pragma unroll
  for (int x = 1; x < kTreeMergeWaves; ++x) merge_state(M, L, A, sm[x][lane].x, sm[x][lane].y, sa[x][lane]);
  const float inv = 1.f / L;
  uint16_t* orow = p.o + (int64_t)b * p.os0 + (int64_t)(kvh * p.group + g) * p.os1 + (int64_t)i * p.os2;
  *reinterpret_cast<u32x2*>(orow + 8 * cg + 4 * hl) =
      live ? u32x2{E::pack2(A.x * inv, A.y * inv), E::pack2(A.z * inv, A.w * inv)} : u32x2{0u, 0u};
}

TreeGeom tree_geometry(int B, int Hq, int Hk, int N, int D, int ctx_limit, int block_size, DeviceShape dev) {
  TreeGeom g{};
  if (B < 1 || Hq < 1 || Hk < 1 || N < 1 || Hq % Hk || block_size < 1 || ctx_limit < 0 ||
      !(D == 16 || D == 32 || D == 64 || D == 128 || D == 256)) {
    g.err = "invalid shape";
    return g;
  }
  if (N > kTreeMaxNodes) {
    g.err = "more than 1024 nodes";
    return g;
  }
  const int64_t rows = (int64_t)(Hq / Hk) * N;
  if (rows > 1 << 24) {
    g.err = "problem too large for one launch";
    return g;
  }
  g.R = (int)rows;
  g.G32 = (g.R + 31) / 32;
  g.QT = std::min(g.R <= 32 ? 1 : g.R <= 64 ? 2 : g.R <= 128 ? 4 : 8, D == 256 ? 4 : 8);
  g.HG = 1;
  for (int h = 2; h * g.QT * 64 <= tree_threads(D, g.QT); h *= 2)
    if (Hk % h == 0 && h * D <= 256) g.HG = h;
  g.NG = Hk / g.HG;
  g.NRT = (g.R + 32 * g.QT - 1) / (32 * g.QT);
  g.NCH = g.HG * D / 8;
  const size_t stage = (size_t)2 * kPagedTile * g.NCH * 16;
  // One workgroup per CU with a ring of 128 KiB, eight stages at most: 32 trees of 16
  // nodes over 256-4096 tokens 40.5 us, 48 with 96 KiB (three 32 KiB stages), 48 and 41
  // with two workgroups of 64 KiB and stages of 32 and 16.
  g.NST = std::min(8, std::max(3, (int)((size_t)128 * 1024 / stage)));
  const int cpt = 2 * (D / (16 * std::min(g.QT, D / 16)));  // copies of an issuing wave per tile
  g.NST = std::min(g.NST, 3 + 63 / cpt);                    // copies of NST - 3 tiles fit vmcnt (see tree_wait)
  // nor more stages than the longest sequence has tiles (and those that reach leaves
  // free): short ones then share a CU
  const int64_t most = (ctx_limit + kPagedTile - 1) / kPagedTile + (g.QT == 8 ? 2 : 1);
  g.NST = (int)std::min<int64_t>(g.NST, std::max<int64_t>(most, 2));
  // behind the ring: block ids, keys whose V is not finite, mask bits of the tiles past
  // the history (34 KiB for 1024 nodes, two stages less)
  const size_t behind = sizeof(int32_t) * (kTreeIds + g.HG * kTreeOddWords + (size_t)(N / 32 + 2) * 32 * g.QT);
  while (g.NST > 3 && (size_t)g.NST * stage + behind > kPagedLdsBudget) --g.NST;
  g.lds_bytes = (size_t)g.NST * stage + behind;
  const int64_t nt_max = (int64_t)B * ((ctx_limit + kPagedTile - 1) / kPagedTile);
  // tiles whose block ids the workgroup can stage
  const int64_t ccap = std::max<int64_t>(1, ((int64_t)(kTreeIds - 2) * block_size) / kPagedTile);
  // Pieces beyond one per sequence, by W = B * per_piece, the workgroups of whole
  // sequences:
  //   2 W <= CUs: as many as fill the CUs once, one workgroup each, of two tiles at least
  //     (1 x 8 nodes over 777 tokens 12.0 us; of one tile 12.3, of four 13.5);
  //   above: as many as there are sequences, so that only those of more tiles than the
  //     average are cut, as a piece pays for its start, the time of some six tiles, and
  //     for its partial states; and none of 32 tiles or fewer while every workgroup has a
  //     CU (10 of 11 nodes over 132-2112 tokens 50 us; none of 64 68, of 8 51), of 64
  //     when they come in rounds (48 of 26 over 1000-2000 58; of 32 70).
  // Against two to four pieces of two tiles or more for every sequence the second rule
  // wins much where sequences are short or rows are many (41 of 110 over 33 tokens
  // 68 -> 30, 22 of 64 over 900 87 -> 42, 17 of 200 over 300-4000 378 -> 256, 48 of 8 over
  // 4000 158 -> 133) and loses a little where few rows read long ragged histories (33
  // of 16 over 500-8000 108 -> 119, 48 of 26 over 2000-4000 126 -> 134). All with P in one
  // part, as the ring's figures above.
  const int64_t per_piece = (int64_t)g.NG * g.NRT;
  const bool busy = 2 * B * per_piece > dev.cus;
  int64_t extra = busy ? B : std::max<int64_t>(1, dev.cus / per_piece - B);
  g.cmin = (int)std::min<int64_t>(ccap, !busy ? 2 : B * per_piece > dev.cus ? 64 : 32);
  extra = std::min(extra, std::max<int64_t>(1, (nt_max + g.cmin - 1) / g.cmin));
  extra = std::max(extra, (nt_max + ccap - 1) / ccap);
  if (extra > INT_MAX / 2) {
    g.err = "problem too large for one launch";
    return g;
  }
  g.extra = (int)extra;
  const int64_t pieces = B + extra;
  const int64_t units = pieces * g.NG;
  const int64_t nx = (int64_t)1 << dev.xcd_shift;
  const int64_t wgs = g.NRT > 1 ? (units + nx - 1) / nx * nx * g.NRT : units;
  // (a grid dimension holds less than 2^32 threads)
  if (wgs * (64 * g.HG * g.QT) > UINT_MAX || B > 65535 ||
      (int64_t)Hk * g.G32 * (D / 8) * (64 * kTreeMergeWaves) > UINT_MAX) {
    g.err = "problem too large for one launch";
    return g;
  }
  g.wgs = (int)wgs;
  // no sequence can have more than one piece when the longest has at most cmin tiles
  g.split = (ctx_limit + kPagedTile - 1) / kPagedTile > g.cmin;
  if (g.split) {
    const size_t slots = (size_t)pieces * Hk * g.G32 * 32;
    g.info_bytes = ((size_t)B * sizeof(int2) + 255) / 256 * 256;
    g.ml_bytes = (slots * sizeof(float2) + 255) / 256 * 256;
    g.part_bytes = slots * D * sizeof(float);
  }
  g.ok = 1;
  return g;
}

template <int DTYPE, int D, int QT>
static hipError_t launch_tree_k(const TreeParams& p, const TreeGeom& g, hipStream_t stream) {
  const hipError_t attr = set_dynamic_lds(reinterpret_cast<const void*>(&tree_fwd_kernel<DTYPE, D, QT>), kPagedLdsBudget);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((tree_fwd_kernel<DTYPE, D, QT>), dim3((unsigned)g.wgs), dim3(64 * g.HG * QT), g.lds_bytes, stream, p);
  return hipGetLastError();
}

template <int DTYPE, int D>
static hipError_t launch_tree_d(const TreeParams& p, const TreeGeom& g, hipStream_t stream) {
  hipError_t e;
  if (p.kn) {
    const unsigned items = (unsigned)p.N * p.updiv.d;
    hipLaunchKernelGGL((tree_append_kernel<DTYPE>), dim3((items + 255) / 256, (unsigned)p.B), dim3(256), 0, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (g.QT == 1) e = launch_tree_k<DTYPE, D, 1>(p, g, stream);
  else if (g.QT == 2) e = launch_tree_k<DTYPE, D, 2>(p, g, stream);
  else if (g.QT == 4) e = launch_tree_k<DTYPE, D, 4>(p, g, stream);
  else {
    if constexpr (D <= 128) e = launch_tree_k<DTYPE, D, 8>(p, g, stream);
    else return hipErrorInvalidValue;
  }
  if (e != hipSuccess || !g.split) return e;
  hipLaunchKernelGGL((tree_merge_kernel<DTYPE, D>), dim3((unsigned)(p.Hk * p.G32 * (D / 8)), (unsigned)p.B),
                     dim3(64 * kTreeMergeWaves), 0, stream, p);
  return hipGetLastError();
}

template <int DTYPE>
static hipError_t launch_tree_t(const TreeParams& p, const TreeGeom& g, int D, hipStream_t stream) {
  switch (D) {
    case 16: return launch_tree_d<DTYPE, 16>(p, g, stream);
    case 32: return launch_tree_d<DTYPE, 32>(p, g, stream);
    case 64: return launch_tree_d<DTYPE, 64>(p, g, stream);
    case 128: return launch_tree_d<DTYPE, 128>(p, g, stream);
    case 256: return launch_tree_d<DTYPE, 256>(p, g, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_tree(const TreeParams& p, const TreeGeom& g, int dtype, int D, hipStream_t stream) {
  return dtype == 0 ? launch_tree_t<0>(p, g, D, stream) : launch_tree_t<1>(p, g, D, stream);
}

}  // namespace cie
