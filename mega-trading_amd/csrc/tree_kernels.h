// gfx950 kernels for generation over a tree of drafted tokens: RoPE by tree
// position, attention of the tree's nodes over a KV cache, and the write of the
// accepted nodes into the caches.
//
// A sequence's tree has N <= 64 nodes; parents[n] is an earlier node or -1 (a
// root: the nodes right behind the cached prefix).  Any other parent, and any
// node below such a one, is padding: its rows are zeros and no node sees it.  A
// node's ancestors (itself included) are one 64-bit word; a wave finds all 64
// words in six rounds of pointer doubling over its lanes, so a chain of 64 costs
// no more than a bush.
#pragma once

#include "attn_kernels.h"
#include "storage.h"

namespace mt {

constexpr int kTreeNodes = 64;  // nodes of a tree: the lanes of a wave, the bits of an ancestor word

struct TreeShape {
  const int* parents;  // [N], int64 stride between sequences (0: one tree for all)
  int64_t parents_stride;
  const int* length_dev;  // cached tokens of each sequence (stride 0 or 1), or null
  int length_stride;
  int length;  // when length_dev is null
  int capacity;
  int N;

  __device__ __forceinline__ int cached(int b) const {
    const int n = length_dev ? length_dev[(int64_t)b * length_stride] : length;
    return min(max(n, 0), capacity);
  }
};

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int src) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x, src, 64), hi = (uint32_t)__shfl((int)(uint32_t)(x >> 32), src, 64);
  return ((uint64_t)hi << 32) | lo;
}

// Lane n: the parent of node n, -2 past the nodes.
__device__ __forceinline__ int tree_parent(const TreeShape& t, int b, int lane) {
  return lane < t.N ? t.parents[(int64_t)b * t.parents_stride + lane] : -2;
}

// Lane n, with its parent: the ancestors of node n and n itself, bit by bit; 0 for padding and for lanes
// past N.  As many rounds as the deepest node asks for: 3 for a chain of 5.
__device__ __forceinline__ uint64_t tree_ancestors(int p, int lane) {
  uint64_t seen = 1ull << lane;
  int up = p >= 0 && p < lane ? p : -1, bad = p != -1 && up < 0;
  while (__ballot(up >= 0)) {
    const int src = up < 0 ? lane : up;
    const uint64_t s = shfl64(seen, src);
    const int b2 = __shfl(bad, src, 64), u2 = __shfl(up, src, 64);
    if (up >= 0) {
      seen |= s;
      bad |= b2;
      up = u2;
    }
  }
  return bad ? 0ull : seen;
}

// ===========================================================================
// RoPE: node n of sequence b is rotated by position cached(b) + depth(n), where
// depth is the number of its ancestors.  q [B, Hq, N, D] and k [B, Hkv, N, D] in
// one launch, one thread per 8 values; fp32 arithmetic, one rounding.  Every
// workgroup finds its sequence's positions itself.  Bound by memory, or by the
// launch: 64 trees of 64 nodes, 40 heads of 128 in fp32 (168 MB) 29 to 34 us (5.0 to
// 5.8 TB/s), 32 trees of 16 nodes, 10 heads of 64 in bf16 3.3 us.
// ===========================================================================
struct TreeRopeParams {
  const void* src[2];
  void* dst[2];      // contiguous [B, H, N, D]
  int64_t s[2][3];   // strides (b, h, n)
  int heads[2];
  TreeShape t;
  const float* cos;  // [table_rows, D/2]
  const float* sin;
  int table_rows, D;
  int blocks;        // workgroups of a sequence
};

template <int DT>
__global__ __launch_bounds__(256) void tree_rope_kernel(TreeRopeParams p) {
  __shared__ int pos[kTreeNodes];
  const int b = blockIdx.x / p.blocks, tid = threadIdx.x;
  if (tid < 64) {
    const uint64_t seen = tree_ancestors(tree_parent(p.t, b, tid), tid);
    pos[tid] = seen ? min(p.t.cached(b) + __popcll(seen) - 1, p.table_rows - 1) : -1;
  }
  __syncthreads();
  const int nc = p.D / 8, N = p.t.N;
  int i = (blockIdx.x % p.blocks) * 256 + tid;
  if (i >= (p.heads[0] + p.heads[1]) * N * nc) return;
  const int c = i % nc;
  i /= nc;
  const int n = i % N;
  i /= N;
  const int w = i >= p.heads[0], h = w ? i - p.heads[0] : i;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (pos[n] >= 0) {
    ops::IO<DT>::load8(p.src[w], b * p.s[w][0] + (int64_t)h * p.s[w][1] + (int64_t)n * p.s[w][2] + 8 * c, x);
    const f32x4 cs = *reinterpret_cast<const f32x4*>(p.cos + (int64_t)pos[n] * (p.D / 2) + 4 * c);
    const f32x4 sn = *reinterpret_cast<const f32x4*>(p.sin + (int64_t)pos[n] * (p.D / 2) + 4 * c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = x[2 * j], o = x[2 * j + 1];
      x[2 * j] = e * cs[j] - o * sn[j];
      x[2 * j + 1] = e * sn[j] + o * cs[j];
    }
  }
  ops::IO<DT>::store8(p.dst[w], (((int64_t)b * p.heads[w] + h) * N + n) * p.D + 8 * c, x);
}

// ===========================================================================
// Attention of the nodes over the cached prefix and their ancestors.
//
// The R N query rows of a KV head (R query heads a group) share its keys.  S^T = K Q^T
// puts one query row on a lane and keys on the accumulator slots, so the probabilities
// feed P V as they are.  The running maximum of a row moves only when a probability
// passes 2^kRescaleSlack.  The tree's own keys follow the prefix as further tiles; only
// they and the prefix's last tile are masked.  Spans of keys that several workgroups
// take are joined by tree_combine_kernel.
//
// tree_attn_kernel: 32 rows and a span; its 8 waves (4 at D = 128) split the span, each
// with K / V tiles of 32 keys of its own (wave-private LDS, two buffers filled by
// asynchronous whole-row copies, no barrier in the loop), and merge their (o, m, l) in
// LDS.  Bound by its chain of dependent steps: length and parents, a tile from memory
// for each step of a wave, the merge.  5 nodes on 200 keys, 8 heads of 64: 6.4 us; 32
// trees of 16 nodes on 545 keys: 8.9 us (an empty launch takes about 2).
//
// tree_attn_rows_kernel: up to 256 rows on shared tiles.  16 sequences of 24 nodes on
// 6001 keys, 32 heads over 8 of 128: 74 to 85 us for 347 MB of keys and values (4.1 to
// 4.7 TB/s, bound by memory); 4 of 64 nodes on 15000 keys, 16 heads over 2 of 64, fp16:
// 28 us, 490 TFLOP/s (bound by the softmax beside the products).
// ===========================================================================
struct TreeAttnParams {
  const uint16_t *q, *k, *v;  // nodes: [B, Hq | Hkv, N, D]
  const uint16_t *kc, *vc;    // caches [B, Hkv, capacity, D]
  uint16_t* out;              // contiguous [B, Hq, N, D]
  float* part;                // [B, Hkv, R N, nspan, D + 4] fp32: o, m (log2), l
  int64_t sq[3], sk[3], sv[3], skc[3], svc[3];  // strides (b, h, n | t)
  TreeShape t;
  int B, Hkv, R;
  int nspan;   // workgroups a row block's keys are split over
  int blocks;  // row blocks of a KV head
  int keys, groups;  // of a tile, and key groups of a workgroup
  float scale_log2;
};

constexpr int kTreeKeys = 32;   // keys of a wave's tile
constexpr float kTreeNone = -1e30f;  // offset of a row that has seen no key: finite, so nothing of it turns into NaN

// Key tiles: the prefix's, then the tree's; and how many of them each of the `groups` key groups of a
// span takes.
struct TreeTiles {
  int prefix, all, per, spans;
  __device__ __forceinline__ TreeTiles(int cached, int N, int nspan, int keys, int groups) {
    prefix = (cached + keys - 1) / keys;
    all = prefix + (N + keys - 1) / keys;
    per = (all + groups * nspan - 1) / (groups * nspan);
    spans = (all + groups * per - 1) / (groups * per);  // that hold tiles
  }
};

// 32 rows [row0, row0 + 32) by one wave; rows past T - 1 copy row T - 1.
template <int D>
__device__ __forceinline__ void copy_rows32(char* lds, const uint16_t* src, int64_t stride, int row0, int T, int lane) {
  using TL = Tile<D>;
  constexpr int RPC = 64 / TL::NC;
#pragma unroll
  for (int c = 0; c < 32 / RPC; ++c) {
    const int row = c * RPC + lane / TL::NC, chunk = (lane % TL::NC) ^ TL::swz(row);
    lds_dma16(src + (int64_t)min(row0 + row, T - 1) * stride + chunk * 8, lds_addr(lds) + c * 1024);
  }
}

// Four values (chunk c) of a query row from the W key groups of a workgroup: M = max m_w,
// o = sum_w 2^(m_w - M) o_w, l the same sum of l_w; into the output, or this span's partial.
template <class E, int D, int W, class FM, class FL, class FO>
__device__ __forceinline__ void tree_merge(const TreeAttnParams& p, int pair, int s, int row, int c, FM m, FL l, FO x) {
  const int64_t at = (int64_t)pair * p.R * p.t.N + row;
  float M = m(0), lt = 0.f;
#pragma unroll
  for (int w = 1; w < W; ++w) M = fmaxf(M, m(w));
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float a = exp2_fast(m(w) - M);
    const f32x4 y = x(w);
    lt = __builtin_fmaf(a, l(w), lt);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(a, y[e], o[e]);
  }
  if (p.nspan == 1) {
    const float inv = 1.f / lt;
    u32x2 y = {pack2<E>(o[0] * inv, o[1] * inv), pack2<E>(o[2] * inv, o[3] * inv)};
    if (lt == 0.f) y = u32x2{0u, 0u};
    *reinterpret_cast<u32x2*>(p.out + at * D + 4 * c) = y;
  } else {
    float* dst = p.part + (at * p.nspan + s) * (D + 4);
    *reinterpret_cast<f32x4*>(dst + 4 * c) = o;
    if (c == 0) *reinterpret_cast<f32x2*>(dst + D) = f32x2{M, lt};
  }
}

// Whether one of the 8 values is infinite or NaN.
template <class E>
__device__ __forceinline__ bool not_finite(u32x4 x) {
  constexpr uint32_t M = std::is_same<E, BF16>::value ? 0x7f80u : 0x7c00u;
  bool r = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (x[i] & M) == M || (x[i] >> 16 & M) == M;
  return r;
}

// The rows of a tile of nodes, one row after the other over NC lanes each (chunk x, taken or not): which of them
// hold a value that is no number, bit by bit; and whether this lane's row does.
template <class E, int NC>
__device__ __forceinline__ uint32_t odd_rows(u32x4 x, bool taken, int lane, bool& mine) {
  const uint64_t bad = __ballot(taken && not_finite<E>(x));
  constexpr uint64_t ROW = (1ull << NC) - 1;
  mine = (bad >> (lane / NC * NC) & ROW) != 0;
  uint32_t rows = 0u;
  if (bad)
#pragma unroll
    for (int r = 0; r < 64 / NC; ++r) rows |= (bad >> (r * NC) & ROW) ? 1u << r : 0u;
  return rows;
}

// A node's values that are no numbers reach its descendants alone: in the tiles, where every row multiplies
// them, 0 stands for all of its values, and the rows that see it (query row `row`) add them here, by the formula.
template <class E, int D>
__device__ __forceinline__ void tree_add_odd(const TreeAttnParams& p, uint64_t odd, uint64_t seen, int b, int kvh, int row,
                                             int hh, float m, f32x16 (&o)[D / 32]) {
  const int rc = min(row, p.R * p.t.N - 1);
  const uint16_t* q = p.q + b * p.sq[0] + (int64_t)(kvh * p.R + rc / p.t.N) * p.sq[1] + (int64_t)(rc % p.t.N) * p.sq[2] + 8 * hh;
  const uint16_t* k = p.k + b * p.sk[0] + (int64_t)kvh * p.sk[1] + 8 * hh;
  const uint16_t* v = p.v + b * p.sv[0] + (int64_t)kvh * p.sv[1] + 4 * hh;
  for (; odd; odd &= odd - 1) {
    const int n = __builtin_ctzll(odd);
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(q + 16 * kk), y = *reinterpret_cast<const u32x4*>(k + n * p.sk[2] + 16 * kk);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = E::dot2(x[e], y[e], s);
    }
    s = sum_with_partner(s);
    if (!(seen >> n & 1)) continue;
    const float w = exp2_fast(__builtin_fmaf(s, p.scale_log2, -m));
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(v + n * p.sv[2] + 32 * dt + 8 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[dt][4 * i + e] = __builtin_fmaf(w, E::to_f((uint16_t)(x[e / 2] >> (16 * (e % 2)))), o[dt][4 * i + e]);
      }
  }
}

template <int D>
constexpr int tree_few_waves() { return D == 128 ? 4 : 8; }  // what the tiles leave room for: one workgroup a CU

template <class E, int D>
__global__ __launch_bounds__(64 * tree_few_waves<D>()) void tree_attn_kernel(TreeAttnParams p) {
  constexpr int W = tree_few_waves<D>();
  using V8 = typename E::v8;
  using TL = Tile<D>;
  constexpr int KT = D / 16, DT = D / 32, TILE = kTreeKeys * TL::RB;
  constexpr int COPIES = 2 * TILE / 1024;  // of a K and a V tile
  constexpr int C4 = D / 4;                // 16-byte chunks of an fp32 row
  __shared__ __attribute__((aligned(1024))) char smem[W][2][2][TILE];  // then the waves' o [32][D] fp32
  __shared__ float wm[W][32], wl[W][32];
  static_assert(sizeof(smem[0]) >= 32 * D * 4, "a wave's o fits its tiles");
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the row blocks of one (sequence, KV head, span) on one XCD (index mod 8), one after the other
  const int slot = blockIdx.x % (8 * p.blocks), g = blockIdx.x / (8 * p.blocks) * 8 + slot % 8, rb = slot / 8;
  if (g >= p.B * p.Hkv * p.nspan) return;
  const int s = g % p.nspan, pair = g / p.nspan, kvh = pair % p.Hkv, b = pair / p.Hkv;
  const int N = p.t.N, RN = p.R * N;
  // the loads that nothing is needed for, together: parents, length and queries
  const int up = tree_parent(p.t, b, lane);
  const int row = rb * 32 + l32, rc = min(row, RN - 1), node = rc % N;
  u32x4 qraw[KT];
  {
    const uint16_t* qr = p.q + b * p.sq[0] + (int64_t)(kvh * p.R + rc / N) * p.sq[1] + (int64_t)node * p.sq[2] + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) qraw[kk] = *reinterpret_cast<const u32x4*>(qr + 16 * kk);
  }
  const int L = p.t.cached(b);
  const TreeTiles tl(L, N, p.nspan, kTreeKeys, W);
  if (s >= tl.spans) return;  // the combine does not read this span
  const int t0 = (s * W + wave) * tl.per, t1 = min(tl.all, t0 + tl.per);

  const uint16_t* kc = p.kc + b * p.skc[0] + (int64_t)kvh * p.skc[1];
  const uint16_t* vc = p.vc + b * p.svc[0] + (int64_t)kvh * p.svc[1];
  const uint16_t* kn = p.k + b * p.sk[0] + (int64_t)kvh * p.sk[1];
  const uint16_t* vn = p.v + b * p.sv[0] + (int64_t)kvh * p.sv[1];
  auto stage = [&](int t, int buf) {
    char *kl = smem[wave][buf][0], *vl = smem[wave][buf][1];
    if (t < tl.prefix) {
      copy_rows32<D>(kl, kc, p.skc[2], t * kTreeKeys, L, lane);
      copy_rows32<D>(vl, vc, p.svc[2], t * kTreeKeys, L, lane);
    } else {
      copy_rows32<D>(kl, kn, p.sk[2], (t - tl.prefix) * kTreeKeys, N, lane);
      copy_rows32<D>(vl, vn, p.sv[2], (t - tl.prefix) * kTreeKeys, N, lane);
    }
  };

  // what the rows see of the tree, and their queries (B operands)
  const uint64_t anc = tree_ancestors(up, lane), above = shfl64(anc, node), seen = row < RN ? above : 0ull;
  V8 qop[KT];
#pragma unroll
  for (int kk = 0; kk < KT; ++kk) qop[kk] = __builtin_bit_cast(V8, seen ? qraw[kk] : zero4());
  const uint64_t padding = ~__ballot(anc != 0ull);  // nodes whose keys and values are not read

  f32x16 oacc[DT];
  float mrun = kTreeNone, lrun = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) zero16(oacc[dt]);
  const int rbase = TL::row_base(lane);
  const TrBase tbase = TL::tr_base(lane);
  const float c2 = p.scale_log2;
  uint64_t odd = 0ull;  // nodes with a value that is no number

  if (t0 < t1) stage(t0, 0);
  if (t0 + 1 < t1) stage(t0 + 1, 1);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    char *kl = smem[wave][buf][0], *vl = smem[wave][buf][1];
    if (t + 1 < t1) copies_done<COPIES>();
    else copies_done<0>();
    const int n0 = (t - tl.prefix) * kTreeKeys;  // the tile's first node, from 0 on
    if (n0 >= 0) {
      // values of padding may be anything, and 0 times it must be 0
#pragma unroll
      for (int i = 0; i < TL::NC / 2; ++i) {
        char* at = vl + (i * 64 + lane) * 16;
        const bool pad = padding >> (n0 + (i * 64 + lane) / TL::NC) & 1;
        bool mine;
        odd |= (uint64_t)odd_rows<E, TL::NC>(*reinterpret_cast<const u32x4*>(at), !pad, lane, mine) << (n0 + i * (64 / TL::NC));
        if (pad || mine) *reinterpret_cast<u32x4*>(at) = zero4();
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    f32x16 st;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk)
      st = E::mfma(TL::template row_op<E>(kl, rbase, 0, kk), qop[kk], kk == 0 ? f32x16{} : st);
    if (n0 >= 0 || (t + 1) * kTreeKeys > L) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i >> 2) + 4 * hh + (i & 3);
        const bool in = n0 >= 0 ? (seen >> (n0 + key)) & 1 : t * kTreeKeys + key < L;
        st[i] = in ? st[i] : -INFINITY;
      }
    }
    V8 pk[2];
    float qs;
    // P = 2^(S c2 - m) in 16 bits; the sums add the rounded values, the weights that P V uses
    auto ex = [&]() {
      u32x4 w[2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2][i & 3] = pack2<E>(exp2_fast(__builtin_fmaf(st[2 * i], c2, -mrun)),
                                    exp2_fast(__builtin_fmaf(st[2 * i + 1], c2, -mrun)));
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s0 = E::sum2(w[0][i], s0);
        s1 = E::sum2(w[1][i], s1);
      }
      qs = s0 + s1;
      pk[0] = __builtin_bit_cast(V8, w[0]);
      pk[1] = __builtin_bit_cast(V8, w[1]);
    };
    ex();
    // a P above 2^kRescaleSlack (or the first keys): that row's m is raised to its maximum.  Other
    // rows of the wave keep theirs, so a row's result does not depend on the rows beside it.
    if (__builtin_amdgcn_ballot_w64(!(qs <= kSumLimit))) {
      float v = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) v = fmaxf(v, st[i]);
      const bool raise = max_with_partner(qs <= kSumLimit ? 0.f : 1.f) > 0.f;
      v = max_with_partner(v) * c2;
      const float m = raise ? fmaxf(mrun, v) : mrun, alpha = exp2_fast(mrun - m);
      mrun = m;
      lrun *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[dt][i] *= alpha;
      ex();
    }
    lrun += qs;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) oacc[dt] = E::mfma(TL::template tr_op<E>(vl, tbase, k2, dt), pk[k2], oacc[dt]);
    if (t + 2 < t1) {
      reads_done();
      stage(t + 2, buf);
    }
  }
  reads_done();
  if (odd) tree_add_odd<E, D>(p, odd, seen, b, kvh, row, hh, mrun, oacc);

  // the wave's o, 16-byte chunk c of row r at slot c ^ (r mod C4)
  float* ow = reinterpret_cast<float*>(smem[wave]);
  const float l = sum_with_partner(lrun);
  if (hh == 0) {
    wm[wave][l32] = seen ? mrun : kTreeNone;
    wl[wave][l32] = seen ? l : 0.f;  // padding: no weight anywhere
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = dt * 8 + 2 * q + hh;
      *reinterpret_cast<f32x4*>(ow + l32 * D + 4 * (c ^ (l32 % C4))) =
          f32x4{oacc[dt][4 * q], oacc[dt][4 * q + 1], oacc[dt][4 * q + 2], oacc[dt][4 * q + 3]};
    }
  __syncthreads();
  for (int i = tid; i < 32 * C4; i += 64 * W) {
    const int r = i / C4, c = i % C4, at = rb * 32 + r;
    if (at >= RN) continue;
    tree_merge<E, D, W>(p, pair, s, at, c, [&](int w) { return wm[w][r]; }, [&](int w) { return wl[w][r]; },
                        [&](int w) {
                          return *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem[w]) + r * D +
                                                                 4 * (c ^ (r % C4)));
                        });
  }
}

// Many query rows: W waves of 32 rows, RW of them on one key tile of 16 RW keys, so that a tile in
// LDS feeds up to 32 RW rows; W / RW key groups, 16 W keys a step in all.  Two buffers; every wave copies 16 rows
// of its group's next tile while it works on the present one, and one barrier a step orders both.
// Two waves a SIMD (four at D <= 64) let one's softmax run beside the other's products.
// (D = 64, 64 KV heads of 256 rows on 10000 keys: 16 waves on tiles of 16 RW keys 61.6 us, 8 on tiles of
// 32 RW keys 76.3; 8 of 512 rows on 15000 keys, join included: 34.4 and 37.6.)
template <int D>
constexpr int tree_waves() { return D == 128 ? 8 : 16; }  // what the tiles leave room for: one workgroup a CU

template <class E, int D, int RW>
__global__ __launch_bounds__(64 * tree_waves<D>()) void tree_attn_rows_kernel(TreeAttnParams p) {
  using V8 = typename E::v8;
  using TL = Tile<D>;
  constexpr int KT = D / 16, DT = D / 32, C4 = D / 4, W = tree_waves<D>();
  constexpr int KEYS = 16 * RW, KW = W / RW, TILE = KEYS * TL::RB, NQ = KEYS / 32;
  constexpr bool AHEAD = D == 128;  // a quarter's scores beside the last one's softmax; else other waves' are
  __shared__ __attribute__((aligned(1024))) char smem[2][KW][2][TILE];  // then the waves' o [32][D] fp32
  __shared__ float wm[W][32], wl[W][32];
  __shared__ uint32_t odd_lds[kTreeNodes / 16];  // nodes with a value that is no number, 16 a word
  static_assert(sizeof(smem) == W * 32 * D * 4, "the waves' o fill the tiles");
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave / RW, rw = wave % RW;
  const int slot = blockIdx.x % (8 * p.blocks), g = blockIdx.x / (8 * p.blocks) * 8 + slot % 8, rb = slot / 8;
  if (g >= p.B * p.Hkv * p.nspan) return;
  const int s = g % p.nspan, pair = g / p.nspan, kvh = pair % p.Hkv, b = pair / p.Hkv;
  const int N = p.t.N, RN = p.R * N;
  const int up = tree_parent(p.t, b, lane);
  const int row = (rb * RW + rw) * 32 + l32, rc = min(row, RN - 1), node = rc % N;
  const bool active = (rb * RW + rw) * 32 < RN;  // wave-uniform
  u32x4 qraw[KT];
  {
    const uint16_t* qr = p.q + b * p.sq[0] + (int64_t)(kvh * p.R + rc / N) * p.sq[1] + (int64_t)node * p.sq[2] + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) qraw[kk] = *reinterpret_cast<const u32x4*>(qr + 16 * kk);
  }
  const int L = p.t.cached(b);
  const TreeTiles tl(L, N, p.nspan, KEYS, KW);
  if (s >= tl.spans) return;  // the combine does not read this span
  const int steps = min(tl.per, (tl.all - s * KW * tl.per + KW - 1) / KW);
  const int first = s * KW * tl.per + kw;  // the group's tiles: first + KW i

  const uint16_t* kc = p.kc + b * p.skc[0] + (int64_t)kvh * p.skc[1];
  const uint16_t* vc = p.vc + b * p.svc[0] + (int64_t)kvh * p.svc[1];
  const uint16_t* kn = p.k + b * p.sk[0] + (int64_t)kvh * p.sk[1];
  const uint16_t* vn = p.v + b * p.sv[0] + (int64_t)kvh * p.sv[1];
  const uint64_t anc = tree_ancestors(up, lane), above = shfl64(anc, node), seen = row < RN ? above : 0ull;
  const uint64_t padding = ~__ballot(anc != 0ull);
  WaveStager<uint16_t, D, 16> ks, vs;
  ks.init(p.skc[2], lane);
  vs.init(p.svc[2], lane);
  // the wave's 16 rows of its group's tile t
  auto stage = [&](int t, int buf) {
    if (t >= tl.all) return;
    char *kl = smem[buf][kw][0] + rw * 16 * TL::RB, *vl = smem[buf][kw][1] + rw * 16 * TL::RB;
    if (t < tl.prefix) {
      ks.stage(kl, kc, p.skc[2], t * KEYS + rw * 16, L);
      vs.stage(vl, vc, p.svc[2], t * KEYS + rw * 16, L);
    } else {
      // the tree's, through registers: what padding holds is replaced by zeros, since 0 times it must be 0
      const int n0 = (t - tl.prefix) * KEYS + rw * 16;
      uint32_t odd = 0u;
#pragma unroll
      for (int i = 0; i < TL::NC / 4; ++i) {
        const int f = i * 64 + lane, row = f / TL::NC, chunk = (f % TL::NC) ^ TL::swz(row), n = n0 + row;
        const bool in = n < N && !(padding >> (n & 63) & 1);
        const u32x4 a = *reinterpret_cast<const u32x4*>(kn + (int64_t)min(n, N - 1) * p.sk[2] + chunk * 8);
        const u32x4 c = *reinterpret_cast<const u32x4*>(vn + (int64_t)min(n, N - 1) * p.sv[2] + chunk * 8);
        bool mine;
        odd |= odd_rows<E, TL::NC>(c, in, lane, mine) << (i * (64 / TL::NC));
        *reinterpret_cast<u32x4*>(kl + f * 16) = in ? a : zero4();
        *reinterpret_cast<u32x4*>(vl + f * 16) = in && !mine ? c : zero4();
      }
      if (n0 < kTreeNodes && lane == 0) odd_lds[n0 / 16] = odd;
    }
  };
  stage(first, 0);
  V8 qop[KT];
#pragma unroll
  for (int kk = 0; kk < KT; ++kk) qop[kk] = __builtin_bit_cast(V8, seen ? qraw[kk] : zero4());
  f32x16 oacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) zero16(oacc[dt]);
  float mrun = kTreeNone, lrun = 0.f;
  const int rbase = TL::row_base(lane);
  const TrBase tbase = TL::tr_base(lane);
  const float c2 = p.scale_log2;
  uint64_t nodes = 0ull;  // of the group's tiles

  for (int i = 0; i < steps; ++i) {
    const int t = first + KW * i, buf = i & 1;
    wait_vmem();
    __syncthreads();  // this step's tiles are there, and the last step's are read
    if (i + 1 < steps) stage(t + KW, buf ^ 1);
    if (!active || t >= tl.all) continue;
    const char *kl = smem[buf][kw][0], *vl = smem[buf][kw][1];
    const int n0 = (t - tl.prefix) * KEYS;  // the tile's first node, from 0 on
    const bool mask = n0 >= 0 || (t + 1) * KEYS > L;
    if (n0 >= 0 && n0 < kTreeNodes) nodes |= (KEYS < 64 ? (1ull << (KEYS % 64)) - 1 : ~0ull) << n0;
    f32x16 st[AHEAD ? 2 : 1];
    auto scores = [&](int h, f32x16& x) {
#pragma unroll
      for (int kk = 0; kk < KT; ++kk)
        x = E::mfma(TL::template row_op<E>(kl, rbase, 32 * h, kk), qop[kk], kk == 0 ? f32x16{} : x);
    };
    if (AHEAD) scores(0, st[0]);
#pragma unroll
    for (int h = 0; h < NQ; ++h) {
      f32x16& x = st[AHEAD ? h & 1 : 0];
      if (!AHEAD) scores(h, x);
      else if (h + 1 < NQ) scores(h + 1, st[(h + 1) & 1]);
      if (mask) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int key = 32 * h + 8 * (j >> 2) + 4 * hh + (j & 3), n = n0 + key;
          const bool in = n0 >= 0 ? n < 64 && (seen >> (n & 63) & 1) : t * KEYS + key < L;
          x[j] = in ? x[j] : -INFINITY;
        }
      }
      V8 pk[2];
      float qs;
      auto ex = [&]() {  // as in tree_attn_kernel
        u32x4 w[2];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j >> 2][j & 3] = pack2<E>(exp2_fast(__builtin_fmaf(x[2 * j], c2, -mrun)),
                                      exp2_fast(__builtin_fmaf(x[2 * j + 1], c2, -mrun)));
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s0 = E::sum2(w[0][j], s0);
          s1 = E::sum2(w[1][j], s1);
        }
        qs = s0 + s1;
        pk[0] = __builtin_bit_cast(V8, w[0]);
        pk[1] = __builtin_bit_cast(V8, w[1]);
      };
      ex();
      if (__builtin_amdgcn_ballot_w64(!(qs <= kSumLimit))) {
        float v = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) v = fmaxf(v, x[j]);
        const bool raise = max_with_partner(qs <= kSumLimit ? 0.f : 1.f) > 0.f;
        v = max_with_partner(v) * c2;
        const float m = raise ? fmaxf(mrun, v) : mrun, alpha = exp2_fast(mrun - m);
        mrun = m;
        lrun *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 16; ++j) oacc[dt][j] *= alpha;
        ex();
      }
      lrun += qs;
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          oacc[dt] = E::mfma(TL::template tr_op<E>(vl, tbase, 2 * h + k2, dt), pk[k2], oacc[dt]);
    }
  }
  __syncthreads();
  if (nodes) {
    uint64_t odd = 0ull;
#pragma unroll
    for (int i = 0; i < kTreeNodes / 16; ++i) odd |= (uint64_t)odd_lds[i] << (16 * i);
    odd &= nodes;
    if (odd) tree_add_odd<E, D>(p, odd, seen, b, kvh, row, hh, mrun, oacc);
  }

  float* ow = reinterpret_cast<float*>(&smem[0][0][0][0]) + wave * 32 * D;
  {
    const float l = sum_with_partner(lrun);
    if (hh == 0) {
      wm[wave][l32] = seen ? mrun : kTreeNone;
      wl[wave][l32] = seen ? l : 0.f;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = dt * 8 + 2 * q + hh;
        *reinterpret_cast<f32x4*>(ow + l32 * D + 4 * (c ^ (l32 % C4))) =
            f32x4{oacc[dt][4 * q], oacc[dt][4 * q + 1], oacc[dt][4 * q + 2], oacc[dt][4 * q + 3]};
      }
  }
  __syncthreads();
  for (int i = tid; i < 32 * RW * C4; i += 64 * W) {
    const int r = i / C4, c = i % C4, l = r % 32, w0 = r / 32, at = rb * RW * 32 + r;
    if (at >= RN) continue;
    tree_merge<E, D, KW>(p, pair, s, at, c, [&](int w) { return wm[w * RW + w0][l]; },
                         [&](int w) { return wl[w * RW + w0][l]; }, [&](int w) {
                           return *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(&smem[0][0][0][0]) +
                                                                  (w * RW + w0) * 32 * D + l * D + 4 * (c ^ (l % C4)));
                         });
  }
}

// Joins the spans of each query row: M = max m_s, o = sum_s 2^(m_s - M) o_s over the same sum of
// l_s.  JOIN threads for each 4 values of a row share its spans, 8 of them in flight each, and meet in LDS.
// 2 spans, 12288 rows of 128: 6.6 us; 4 spans, 4096 rows of 64: 4.2.
template <class E, int D, int JOIN>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeAttnParams p) {
  constexpr int C4 = D / 4, ROW = D + 4, BATCH = 8, ROWS = 256 / (C4 * JOIN);
  __shared__ __attribute__((aligned(16))) float part[ROWS][JOIN][ROW];
  const int tid = threadIdx.x, c = tid % C4, j = tid / C4 % JOIN, r = tid / (C4 * JOIN), RN = p.R * p.t.N;
  const int64_t row = min((int64_t)blockIdx.x * ROWS + r, (int64_t)p.B * p.Hkv * RN - 1);  // the last ones twice
  const int b = int(row / ((int64_t)p.Hkv * RN));
  const int ns = TreeTiles(p.t.cached(b), p.t.N, p.nspan, p.keys, p.groups).spans;
  const float* src = p.part + row * p.nspan * ROW;
  float M = kTreeNone, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = j; s0 < ns; s0 += BATCH * JOIN) {
    f32x2 ml[BATCH];
    f32x4 x[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float* q = src + (int64_t)min(s0 + JOIN * i, ns - 1) * ROW;
      ml[i] = *reinterpret_cast<const f32x2*>(q + D);
      x[i] = *reinterpret_cast<const f32x4*>(q + 4 * c);
    }
    float mn = M;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) mn = fmaxf(mn, ml[i][0]);
    const float a = exp2_fast(M - mn);
    l *= a;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (s0 + JOIN * i >= ns) continue;
      const float w = exp2_fast(ml[i][0] - mn);
      l = __builtin_fmaf(w, ml[i][1], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, x[i][e], o[e]);
    }
    M = mn;
  }
  *reinterpret_cast<f32x4*>(&part[r][j][4 * c]) = o;
  if (c == 0) *reinterpret_cast<f32x2*>(&part[r][j][D]) = f32x2{M, l};
  __syncthreads();
  if (j) return;
  float top = kTreeNone, lt = 0.f;
#pragma unroll
  for (int i = 0; i < JOIN; ++i) top = fmaxf(top, part[r][i][D]);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < JOIN; ++i) {
    const float w = exp2_fast(part[r][i][D] - top);
    const f32x4 x = *reinterpret_cast<const f32x4*>(&part[r][i][4 * c]);
    lt = __builtin_fmaf(w, part[r][i][D + 1], lt);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(w, x[e], y[e]);
  }
  const float inv = 1.f / lt;
  u32x2 z = {pack2<E>(y[0] * inv, y[1] * inv), pack2<E>(y[2] * inv, y[3] * inv)};
  if (lt == 0.f) z = u32x2{0u, 0u};
  *reinterpret_cast<u32x2*>(p.out + row * D + 4 * c) = z;
}

// ===========================================================================
// Accepted nodes into the caches: cache[b, h, cached(b) + j] = node[b, h, path[b, j]]
// for j < count[b], keys and values of up to kCommitLayers layers in one launch.  A thread takes W
// 16-bit values of one (layer, key or value, head) and every split-th node, four of them in flight.
// 8 layers, 64 trees with 24 of 64 nodes accepted, 8 heads of 128: 11 to 17 us for 50 MB read and written;
// 32 trees of 16 nodes, 2 heads of 64: 3.4 us, the launch's latency.
// ===========================================================================
constexpr int kCommitLayers = 32;

struct TreeCommitParams {
  const uint16_t* src[2][kCommitLayers];  // [B, Hkv, N, D]: keys, values
  uint16_t* dst[2][kCommitLayers];        // [B, Hkv, capacity, D]
  int64_t ss[2][3], sd[2][3];             // strides (b, h, n | t), one for all layers
  const int *path, *count;                // [B, N], [B]
  TreeShape t;                            // parents unused
  int layers, Hkv, D;
  int split;   // threads that share a (layer, key or value, head, values)
  int blocks;  // workgroups of a sequence
};

template <int W>
__global__ __launch_bounds__(256) void tree_commit_kernel(TreeCommitParams p) {
  using V = typename std::conditional<W == 8, u32x4, uint16_t>::type;
  constexpr int AHEAD = 4;
  const int b = blockIdx.x / p.blocks, nc = p.D / W, N = p.t.N;
  int64_t i = (int64_t)(blockIdx.x % p.blocks) * 256 + threadIdx.x;
  const int c = int(i % nc);
  i /= nc;
  const int h = int(i % p.Hkv);
  i /= p.Hkv;
  const int w = int(i % 2);
  i /= 2;
  const int layer = int(i % p.layers), first = int(i / p.layers);
  if (first >= p.split) return;
  const uint16_t* src = p.src[w][layer] + b * p.ss[w][0] + (int64_t)h * p.ss[w][1] + W * c;
  uint16_t* dst = p.dst[w][layer] + b * p.sd[w][0] + (int64_t)h * p.sd[w][1] + W * c;
  const int cached = p.t.cached(b), count = min(p.count[b], min(N, p.t.capacity - cached));
  for (int j0 = first; j0 < count; j0 += AHEAD * p.split) {
    int node[AHEAD];
    V x[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) node[a] = p.path[(int64_t)b * N + min(j0 + a * p.split, N - 1)];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
      x[a] = *reinterpret_cast<const V*>(src + (int64_t)min(max(node[a], 0), N - 1) * p.ss[w][2]);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int j = j0 + a * p.split;
      if (j < count && node[a] >= 0 && node[a] < N) *reinterpret_cast<V*>(dst + (int64_t)(cached + j) * p.sd[w][2]) = x[a];
    }
  }
}

}  // namespace mt
