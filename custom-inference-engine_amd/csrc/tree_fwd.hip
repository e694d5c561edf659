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
// serves all of them. A wave holds MW groups of 32 rows (one row per lane pair,
// see common.hpp), QT waves side by side cover a row tile of 32 QT MW rows of
// one kv head, and a workgroup takes HG kv heads: HG * QT waves. Rows beyond
// one tile go to workgroups of their own.
//
// Keys. A piece, one workgroup's work, is a run of 32-token tiles of ONE
// sequence. Every workgroup finds its own from the context lengths: with C the
// tiles per piece that spreads all sequences' tiles over the launch's
// workgroups, sequence b has ceil(tiles_b / C) pieces of nearly equal length,
// so ragged batches balance and the host needs no lengths. A sequence of more
// pieces than one leaves partial states (acc, m, l) that tree_merge_kernel
// combines in a fixed order.
//
// Per tile: K and V go global -> LDS by 16-byte direct copies into a ring of NST
// stages (one barrier per tile: the stage refilled after it was read before it),
//   S^T = K Q^T, online softmax in registers, O^T += V^T P^T
// as in paged_fwd.hip. Only tiles that reach past the history look at the tree
// mask: a lane cuts the 32 bits of the tile out of its row's words.
//
// P is rounded to the 16-bit type for the second product, as in the dense and
// paged kernels; its sum is fp32 and of the unrounded values.
//
// A masked key must not reach a row even if its V holds infinities or NaN (the
// slots of padding nodes are never written): in a tile past the history such
// values are taken out of the product and added for the rows that see their key.
#include <climits>

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

template <int PT>
__device__ __forceinline__ void tree_wait(int ahead) {
  // vmcnt counts the PT copies of every tile issued after the one needed
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

template <int DTYPE, int D, int QT, int MW>
__global__ __launch_bounds__(256) void tree_fwd_kernel(const TreeParams p) {
  warm_kernargs<sizeof(TreeParams)>();
  using C = TreeCfg<D, QT>;
  using E = Elt<DTYPE>;
  extern __shared__ __attribute__((aligned(16))) uint16_t ring[];
  __shared__ int32_t sbt[kTreeIds];

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

  // ---- query rows ------------------------------------------------------------
  int node[MW], hq[MW];
  bool rv[MW], live[MW];
  const int32_t* words[MW];
  uint16_t* orow[MW];
#pragma unroll
  for (int m = 0; m < MW; ++m) {
    const int r = ((rt * QT + qt) * MW + m) * 32 + l32;
    rv[m] = r < p.R;
    const int g = rv[m] ? (int)fdiv((uint32_t)r, p.ndiv) : 0;
    node[m] = rv[m] ? r - g * p.N : 0;
    hq[m] = kvh * p.group + g;
    words[m] = p.mask + (int64_t)b * p.ms0 + (int64_t)node[m] * p.ms1;
    orow[m] = p.o + (int64_t)b * p.os0 + hq[m] * p.os1 + (int64_t)node[m] * p.os2;
  }
  if (t == 0) {  // an invalid context length
#pragma unroll
    for (int m = 0; m < MW; ++m)
      if (rv[m]) tree_fill<D>(orow[m], hl, tree_row_live(words[m], p.N) ? nan2 : 0u);
    return;
  }
  const int per_piece = (int)(((uint32_t)t + (uint32_t)n - 1) / (uint32_t)n);
  const int tlo = (j - j0) * per_piece, thi = min(t, tlo + per_piece), T = thi - tlo;
  const int base = ctx - p.N;

  // ---- block ids of the piece ------------------------------------------------
  const int blk_lo = (int)fdiv((uint32_t)(kPagedTile * tlo), p.bsdiv);
  const int nids = (int)fdiv((uint32_t)(min(ctx, kPagedTile * thi) - 1), p.bsdiv) - blk_lo + 1;
  bool bad = false;
  {
    const int32_t* src = p.bt + (int64_t)b * p.max_blocks + blk_lo;
    for (int x = threadIdx.x; x < nids; x += blockDim.x) {
      const int id = src[x];
      const bool ok = (uint32_t)id < (uint32_t)p.num_blocks;
      bad |= !ok;
      sbt[x] = ok ? id : -1;
    }
  }

  u32x4 qf[MW][C::KK];
#pragma unroll
  for (int m = 0; m < MW; ++m) {
    const uint16_t* qrow = p.q + (int64_t)b * p.qs0 + hq[m] * p.qs1 + (int64_t)node[m] * p.qs2;
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) qf[m][kk] = load16(qrow + 16 * kk + 8 * hl, rv[m]);
    live[m] = tree_row_live(words[m], p.N);
  }
  if (p.rope.cos) {
    // node i is rotated at position base + its depth
#pragma unroll
    for (int m = 0; m < MW; ++m)
      rope_q_lane<DTYPE, D>(qf[m], p.rope, base + max(p.depths[(int64_t)b * p.ds0 + node[m]], 0), rv[m], hl);
  }
#pragma unroll
  for (int m = 0; m < MW; ++m)
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) qf[m][kk] ^= u32x4{p.q_sign, p.q_sign, p.q_sign, p.q_sign};
  const bool poison = __syncthreads_or(bad);  // an id outside the pool: NaN rows, never a read

  // ---- copies ----------------------------------------------------------------
  const int NCH = p.NCH, NST = p.NST;
  const int lg_nch = __builtin_ctz(NCH);
  const int TILE_EL = kPagedTile * NCH * 8;
  const int STAGE_EL = 2 * TILE_EL;
  const bool issuer = qt < C::QTI;
  const int c0 = (hh * C::QTI + qt) * C::CPW;  // this wave's first copy of a tensor's tile
  int ltok[C::CPW];
  int32_t goffk[C::CPW], goffv[C::CPW];
#pragma unroll
  for (int x = 0; x < C::CPW; ++x) {
    const int P = 64 * (c0 + x) + lane;
    const int tk = P >> lg_nch;
    const int c = (P & (NCH - 1)) ^ row_swizzle(NCH, tk & (kPagedTile - 1));
    const int hd = c / C::S, dc = c % C::S;
    ltok[x] = tk;
    goffk[x] = (gh * p.HG + hd) * (int32_t)p.ks2 + 8 * dc;
    goffv[x] = (gh * p.HG + hd) * (int32_t)p.vs2 + 8 * dc;
  }
  const uint32_t ring_lds = lds_addr_of(ring);
  int i_stage = 0;
  auto issue = [&](int k) __attribute__((always_inline)) {
    const int tbase = kPagedTile * (tlo + k);
    const uint32_t st = ring_lds + 2u * (uint32_t)(i_stage * STAGE_EL) + 1024u * (uint32_t)c0;
    i_stage = i_stage + 1 == NST ? 0 : i_stage + 1;
    int bid[C::CPW], off[C::CPW];
#pragma unroll
    for (int x = 0; x < C::CPW; ++x) {
      const int tk = min(tbase + ltok[x], ctx - 1);
      const int blk = (int)fdiv((uint32_t)tk, p.bsdiv);
      off[x] = tk - blk * p.block_size;
      bid[x] = max(sbt[blk - blk_lo], 0);
    }
#pragma unroll
    for (int x = 0; x < C::CPW; ++x) {
      dma16_at_nt(p.kc + (int64_t)bid[x] * p.ks0 + (int64_t)off[x] * p.ks1 + goffk[x], st + 1024u * x);
      dma16_at_nt(p.vc + (int64_t)bid[x] * p.vs0 + (int64_t)off[x] * p.vs1 + goffv[x], st + 2u * TILE_EL + 1024u * x);
    }
  };
  if (issuer)
    for (int k = 0; k < min(NST - 1, T); ++k) issue(k);

  // ---- tile loop -------------------------------------------------------------
  const int swk = row_swizzle(NCH, l32);
  const int rq = lane & 15, gq = lane >> 4;
  int swv[2][2];
#pragma unroll
  for (int cc = 0; cc < 2; ++cc) {
    swv[cc][0] = row_swizzle(NCH, 16 * cc + 4 * hl + (rq >> 2));
    swv[cc][1] = row_swizzle(NCH, 16 * cc + 4 * hl + (rq >> 2) + 8);
  }
  f32x16 acc[MW][C::DT];
  float mx[MW], l[MW];
#pragma unroll
  for (int m = 0; m < MW; ++m) {
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) acc[m][dt] = f32x16{};
    mx[m] = -INFINITY;
    l[m] = 0.f;
  }
  const float c = p.scale_log2;
  int c_stage = 0;

  for (int k = 0; k < T; ++k) {
    if (issuer) tree_wait<2 * C::CPW>(min(NST - 2, T - 1 - k));
    __syncthreads();  // tile k is in LDS for every wave, and every wave is done with tile k - 1
    if (issuer && k + NST - 1 < T) issue(k + NST - 1);
    const uint16_t* kst = ring + c_stage * STAGE_EL;
    const uint16_t* vst = kst + TILE_EL;
    c_stage = c_stage + 1 == NST ? 0 : c_stage + 1;
    const int t0 = kPagedTile * (tlo + k);

    f32x16 sc[MW];
#pragma unroll
    for (int m = 0; m < MW; ++m) sc[m] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      const int pos = (hh * C::S + 2 * kk + hl) ^ swk;
      const u32x4 a = *reinterpret_cast<const u32x4*>(kst + ((l32 << lg_nch) + pos) * 8);
#pragma unroll
      for (int m = 0; m < MW; ++m) sc[m] = E::mfma(a, qf[m][kk], sc[m]);
    }
    const bool tail = t0 + kPagedTile > base;
    uint32_t vis[MW], odd_keys = 0;
    bool odd = false;
    if (tail) {
#pragma unroll
      for (int m = 0; m < MW; ++m) {
        vis[m] = tree_bits(words[m], t0 - base, p.N, p.W, live[m]);
        const uint32_t mine = vis[m] >> (4 * hl);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sc[m][e] = (mine >> (8 * (e >> 2) + (e & 3))) & 1u ? sc[m][e] : -INFINITY;
      }
      // keys of this head whose V has a value that is not finite
      odd_keys = 0;
      for (int x = lane; x < kPagedTile * C::S; x += 64) {
        const int tk = x / C::S, cc = (hh * C::S + x % C::S) ^ row_swizzle(NCH, tk);
        const u32x4 v = *reinterpret_cast<const u32x4*>(vst + ((tk << lg_nch) + cc) * 8);
        if (!all_finite<DTYPE>(v)) odd_keys |= 1u << tk;
      }
      odd = __builtin_amdgcn_ballot_w64(odd_keys != 0) != 0;
      if (odd)
        for (int x = 1; x < 64; x *= 2) odd_keys |= (uint32_t)__shfl_xor((int)odd_keys, x);
    }
    u32x4 pb[MW][2];
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      const float mxs = xhalf_max(max16(sc[m])) * c;
      const bool grow = mxs > mx[m] + kLazyRescaleTree;
      if (__builtin_amdgcn_ballot_w64(grow)) {
        const float m_new = grow ? mxs : mx[m];
        const float alpha = grow ? exp2_fast(mx[m] - m_new) : 1.f;
        l[m] *= alpha;
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt) acc[m][dt] *= alpha;
        mx[m] = m_new;
      }
      const float neg_m = mx[m] == -INFINITY ? 0.f : -mx[m];
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[m][e] = exp2_fast(fmaf(sc[m][e], c, neg_m));
      l[m] += sum16(sc[m]);
#pragma unroll
      for (int cc = 0; cc < 2; ++cc)
#pragma unroll
        for (int x = 0; x < 4; ++x) pb[m][cc][x] = E::pack2(sc[m][8 * cc + 2 * x], sc[m][8 * cc + 2 * x + 1]);
    }
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) {
      int d = 32 * dt + 16 * (gq & 1) + 4 * (rq & 3);
      if (D < 32) d = min(d, D - 4);  // rows >= D of O^T are discarded
      const int chunk = hh * C::S + (d >> 3), within = d & 7;
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const int tl = 16 * cc + 4 * hl + (rq >> 2), th = tl + 8;
        const u32x2 lo = lds_read_tr16(vst + ((tl << lg_nch) + (chunk ^ swv[cc][0])) * 8 + within);
        const u32x2 hi = lds_read_tr16(vst + ((th << lg_nch) + (chunk ^ swv[cc][1])) * 8 + within);
        u32x4 a = {lo[0], lo[1], hi[0], hi[1]};
        if (odd) a = finite_or_zero<DTYPE>(a);
#pragma unroll
        for (int m = 0; m < MW; ++m) acc[m][dt] = E::mfma(a, pb[m][cc], acc[m][dt]);
      }
    }
    // the values left out, for the rows that see their key
    for (uint32_t keys = odd ? __builtin_amdgcn_readfirstlane(odd_keys) : 0u; keys; keys &= keys - 1) {
      const int tk = __builtin_ctz(keys), es = 4 * (tk >> 3) + (tk & 3);
      const uint16_t* vrow = vst + (tk << lg_nch) * 8;
      const int sw = row_swizzle(NCH, tk);
#pragma unroll
      for (int m = 0; m < MW; ++m) {
        float pe = sc[m][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) pe = e == es ? sc[m][e] : pe;
        pe = __shfl(pe, l32 + 32 * ((tk >> 2) & 1));
        const bool seen = (vis[m] >> tk) & 1u;
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
          for (int g4 = 0; g4 < 4; ++g4) {
            const int d = 32 * dt + 8 * g4 + 4 * hl;
            if (D < 32 && d >= D) continue;
            const u32x2 v4 = *reinterpret_cast<const u32x2*>(vrow + ((hh * C::S + (d >> 3)) ^ sw) * 8 + (d & 7));
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t h = y & 1 ? v4[y >> 1] >> 16 : v4[y >> 1] & 0xffffu;
              if (seen && (h & kExp<DTYPE>) == kExp<DTYPE>) acc[m][dt][4 * g4 + y] += pe * widen<DTYPE>(h);
            }
          }
      }
    }
  }

  // ---- output ----------------------------------------------------------------
#pragma unroll
  for (int m = 0; m < MW; ++m) {
    const float lt = xhalf_sum(l[m]);
    if (!rv[m]) continue;
    if (n == 1) {
      if (!live[m]) {
        tree_fill<D>(orow[m], hl, 0u);
        continue;
      }
      const float inv = poison ? __builtin_nanf("") : 1.f / lt;
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int d = 32 * dt + 8 * g4 + 4 * hl;
          if (D >= 32 || d < D)
            *reinterpret_cast<u32x2*>(orow[m] + d) =
                u32x2{E::pack2(acc[m][dt][4 * g4] * inv, acc[m][dt][4 * g4 + 1] * inv),
                      E::pack2(acc[m][dt][4 * g4 + 2] * inv, acc[m][dt][4 * g4 + 3] * inv)};
        }
    } else {
      const int r = ((rt * QT + qt) * MW + m) * 32 + l32;
      const int64_t slot = ((int64_t)j * p.Hk + kvh) * p.R + r;
      const float pz = poison ? __builtin_nanf("") : 1.f;
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int d = 32 * dt + 8 * g4 + 4 * hl;
          if (D >= 32 || d < D)
            *reinterpret_cast<float4*>(p.part + slot * D + d) =
                float4{acc[m][dt][4 * g4] * pz, acc[m][dt][4 * g4 + 1] * pz, acc[m][dt][4 * g4 + 2] * pz,
                       acc[m][dt][4 * g4 + 3] * pz};
        }
      if (hl == 0) p.ml[slot] = float2{mx[m] * pz, lt * pz};
    }
  }
}

// Writes the nodes' K and V behind the history before attention reads them:
// node i of sequence b (rows b * N + i of kn / vn) to position base + i, K
// rotated at base + its depth. One thread moves a pair of 16-byte chunks (the
// two halves that a rotation mixes) of K and of V. Padding slots, positions
// outside the rotary tables and invalid sequences are left as they are.
template <int DTYPE>
__global__ __launch_bounds__(256) void tree_append_kernel(const TreeParams p) {
  warm_kernargs<sizeof(TreeParams)>();
  const int b = blockIdx.y;
  const uint32_t x = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = fdiv(x, p.updiv);  // node
  if (row >= (uint32_t)p.N) return;
  const int ctx = p.lens[b];
  const uint32_t c = x - row * p.updiv.d;
  const int half = p.D / 2, h = (int)(c / (uint32_t)(p.D / 16)), d = 8 * (int)(c % (uint32_t)(p.D / 16));
  const int64_t r = (int64_t)b * p.N + row;
  const uint16_t* ks = p.kn + r * p.kns0 + h * p.kns1 + d;
  const uint16_t* vs = p.vn + r * p.vns0 + h * p.vns1 + d;
  u32x4 k0 = *reinterpret_cast<const u32x4*>(ks), k1 = *reinterpret_cast<const u32x4*>(ks + half);
  const u32x4 v0 = *reinterpret_cast<const u32x4*>(vs), v1 = *reinterpret_cast<const u32x4*>(vs + half);
  if (!tree_ctx_valid(p, ctx) || !tree_row_live(p.mask + (int64_t)b * p.ms0 + (int64_t)row * p.ms1, p.N)) return;
  const int pos = ctx - p.N + (int)row;
  const int blk = (int)fdiv((uint32_t)pos, p.bsdiv), off = pos - blk * p.block_size;
  const int id = p.bt[(int64_t)b * p.max_blocks + blk];
  if ((uint32_t)id >= (uint32_t)p.num_blocks) return;
  if (p.rope.cos) {
    const int at = ctx - p.N + max(p.depths[(int64_t)b * p.ds0 + row], 0);
    if (at >= p.rope.rows) return;
    rope_apply8<DTYPE>(k0, k1, rope_load(p.rope, (int64_t)at * half + d), p.rope.dt);
  }
  uint16_t* kd = const_cast<uint16_t*>(p.kc) + (int64_t)id * p.ks0 + (int64_t)off * p.ks1 + (int64_t)h * p.ks2 + d;
  uint16_t* vd = const_cast<uint16_t*>(p.vc) + (int64_t)id * p.vs0 + (int64_t)off * p.vs1 + (int64_t)h * p.vs2 + d;
  *reinterpret_cast<u32x4*>(kd) = k0;
  *reinterpret_cast<u32x4*>(kd + half) = k1;
  *reinterpret_cast<u32x4*>(vd) = v0;
  *reinterpret_cast<u32x4*>(vd + half) = v1;
}

// Combines the pieces of every sequence that has more than one. Eight lanes
// share a row's four columns: lane t takes pieces t, t + 8, ..., then a fixed
// butterfly joins the eight states.
constexpr int kTreeMergeLanes = 8, kTreeMergeBatch = 4;

template <int DTYPE, int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeParams p) {
  using E = Elt<DTYPE>;
  constexpr int Q4 = D / 4;
  warm_kernargs<sizeof(TreeParams)>();
  const int b = blockIdx.y;
  const int2 inf = p.info[b];
  if (inf.y < 2) return;  // written whole by the main pass
  const uint32_t tid = blockIdx.x * 256u + threadIdx.x;
  const int t = (int)(tid % kTreeMergeLanes);
  const uint32_t item = tid / kTreeMergeLanes;
  const int d4 = (int)(item % Q4);
  const uint32_t row = item / Q4;  // kvh * R + r
  const bool in = row < (uint32_t)(p.Hk * p.R);
  float M = -INFINITY, L = 0.f;
  float4 A = {0.f, 0.f, 0.f, 0.f};
  if (in)
    for (int k0 = t; k0 < inf.y; k0 += kTreeMergeLanes * kTreeMergeBatch) {
      float2 ml[kTreeMergeBatch];
      float4 a[kTreeMergeBatch];
#pragma unroll
      for (int u = 0; u < kTreeMergeBatch; ++u) {
        const int k = min(k0 + kTreeMergeLanes * u, inf.y - 1);
        const int64_t slot = (int64_t)(inf.x + k) * p.Hk * p.R + row;
        ml[u] = p.ml[slot];
        a[u] = *reinterpret_cast<const float4*>(p.part + slot * D + 4 * d4);
      }
#pragma unroll
      for (int u = 0; u < kTreeMergeBatch; ++u)
        if (k0 + kTreeMergeLanes * u < inf.y) merge_state(M, L, A, ml[u].x, ml[u].y, a[u]);
    }
  butterfly_step<1>(t, M, L, A);
  butterfly_step<2>(t, M, L, A);
  butterfly_step<4>(t, M, L, A);
  if (!in || t != 0) return;
  const int kvh = (int)(row / (uint32_t)p.R), r = (int)(row - (uint32_t)kvh * (uint32_t)p.R);
  const int g = (int)fdiv((uint32_t)r, p.ndiv), i = r - g * p.N;
  const bool live = tree_row_live(p.mask + (int64_t)b * p.ms0 + (int64_t)i * p.ms1, p.N);
  const float inv = 1.f / L;
  uint16_t* orow = p.o + (int64_t)b * p.os0 + (int64_t)(kvh * p.group + g) * p.os1 + (int64_t)i * p.os2;
  *reinterpret_cast<u32x2*>(orow + 4 * d4) =
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
  if (rows * Hk * (D / 4) * kTreeMergeLanes >= ((int64_t)1 << 31)) {
    g.err = "problem too large for one launch";
    return g;
  }
  g.R = (int)rows;
  g.QT = g.R <= 32 ? 1 : g.R <= 64 ? 2 : 4;
  g.MW = g.R > 128 && D <= 128 ? 2 : 1;
  g.HG = 1;
  for (int h = 2; h <= 4 / g.QT; h *= 2)
    if (Hk % h == 0 && h * D <= 256) g.HG = h;
  g.NG = Hk / g.HG;
  const int rt = 32 * g.QT * g.MW;
  g.NRT = (g.R + rt - 1) / rt;
  g.NCH = g.HG * D / 8;
  const size_t stage = (size_t)2 * kPagedTile * g.NCH * 16;
  g.NST = std::min(4, std::max(2, (int)((size_t)64 * 1024 / stage)));
  const int cpt = 2 * (D / (16 * std::min(g.QT, D / 16)));  // copies of an issuing wave per tile
  g.NST = std::min(g.NST, 2 + 63 / cpt);                    // those of NST - 2 tiles in flight fit vmcnt
  g.lds_bytes = (size_t)g.NST * stage;
  const int wpc = std::max(1, std::min(2, (int)((size_t)150 * 1024 / (g.lds_bytes + sizeof(int32_t) * kTreeIds))));
  const int64_t nt_max = (int64_t)B * ((ctx_limit + kPagedTile - 1) / kPagedTile);
  // tiles whose block ids the workgroup can stage
  const int64_t ccap = std::max<int64_t>(1, ((int64_t)(kTreeIds - 2) * block_size) / kPagedTile);
  const int64_t per_piece = (int64_t)g.NG * g.NRT;
  const int64_t want = ((int64_t)dev.cus * wpc + per_piece - 1) / per_piece;  // pieces that fill the device once
  int64_t extra = std::max<int64_t>(std::max<int64_t>(want - B, want / 2), 1);
  g.cmin = (int)std::min<int64_t>(ccap, g.R <= 64 ? 2 : 4);
  extra = std::min(extra, std::max<int64_t>(1, (nt_max + g.cmin - 1) / g.cmin));
  extra = std::max(extra, (nt_max + ccap - 1) / ccap);
  g.extra = (int)extra;
  const int64_t pieces = B + extra;
  const int64_t units = pieces * g.NG;
  const int64_t nx = (int64_t)1 << dev.xcd_shift;
  const int64_t wgs = g.NRT > 1 ? (units + nx - 1) / nx * nx * g.NRT : units;
  if (wgs > INT_MAX || B > 65535) {
    g.err = "problem too large for one launch";
    return g;
  }
  g.wgs = (int)wgs;
  // no sequence can have more than one piece when the longest has at most cmin tiles
  g.split = (ctx_limit + kPagedTile - 1) / kPagedTile > g.cmin;
  if (g.split) {
    const size_t slots = (size_t)pieces * Hk * g.R;
    g.info_bytes = ((size_t)B * sizeof(int2) + 255) / 256 * 256;
    g.ml_bytes = (slots * sizeof(float2) + 255) / 256 * 256;
    g.part_bytes = slots * D * sizeof(float);
  }
  g.ok = 1;
  return g;
}

template <int DTYPE, int D, int QT, int MW>
static hipError_t launch_tree_k(const TreeParams& p, const TreeGeom& g, hipStream_t stream) {
  const hipError_t attr = set_dynamic_lds(reinterpret_cast<const void*>(&tree_fwd_kernel<DTYPE, D, QT, MW>), kPagedLdsBudget);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((tree_fwd_kernel<DTYPE, D, QT, MW>), dim3((unsigned)g.wgs), dim3(64 * g.HG * QT), g.lds_bytes, stream, p);
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
  if (g.QT == 1) e = launch_tree_k<DTYPE, D, 1, 1>(p, g, stream);
  else if (g.QT == 2) e = launch_tree_k<DTYPE, D, 2, 1>(p, g, stream);
  else if (g.MW == 1) e = launch_tree_k<DTYPE, D, 4, 1>(p, g, stream);
  else {
    if constexpr (D <= 128) e = launch_tree_k<DTYPE, D, 4, 2>(p, g, stream);
    else return hipErrorInvalidValue;
  }
  if (e != hipSuccess || !g.split) return e;
  const unsigned items = (unsigned)(p.Hk * p.R) * (D / 4) * kTreeMergeLanes;
  hipLaunchKernelGGL((tree_merge_kernel<DTYPE, D>), dim3((items + 255) / 256, (unsigned)p.B), dim3(256), 0, stream, p);
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
