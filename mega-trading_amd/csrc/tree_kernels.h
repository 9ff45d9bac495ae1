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

// Lane n: the ancestors of node n and n itself, bit by bit; 0 for padding and for lanes past N.
__device__ __forceinline__ uint64_t tree_ancestors(const TreeShape& t, int b, int lane) {
  const int p = lane < t.N ? t.parents[(int64_t)b * t.parents_stride + lane] : -2;
  uint64_t seen = 1ull << lane;
  int up = p >= 0 && p < lane ? p : -1, bad = p != -1 && up < 0;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
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
// one launch, one thread per 8 values; fp32 arithmetic, one rounding.
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
    const uint64_t seen = tree_ancestors(p.t, b, tid);
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
// The R N query rows of a KV head (R query heads a group) share its keys.  A
// workgroup takes 32 NT of those rows and a span of the keys; its 4 waves split
// the span, each with K / V tiles of 32 keys of its own (wave-private LDS, two
// buffers filled by asynchronous whole-row copies, no barrier in the loop), and
// merge their (o, m, l) in LDS.  Several spans of one row block are joined by
// tree_combine_kernel.  S^T = K Q^T puts one query row on a lane and keys on the
// accumulator slots, so the probabilities feed P V as they are.  The tree's own
// keys follow the prefix as one or two more tiles; only they and the prefix's last
// tile are masked.
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
  float scale_log2;
};

constexpr int kTreeKeys = 32;   // keys of a wave's tile
constexpr int kTreeWaves = 4;
constexpr float kTreeNone = -1e30f;  // offset of a row that has seen no key: finite, so nothing of it turns into NaN

// Tiles of 32 keys: the prefix's, then the tree's; and how many of them a wave takes.
struct TreeTiles {
  int prefix, all, per;
  __device__ __forceinline__ TreeTiles(int cached, int N, int nspan) {
    prefix = (cached + kTreeKeys - 1) / kTreeKeys;
    all = prefix + (N + kTreeKeys - 1) / kTreeKeys;
    per = (all + kTreeWaves * nspan - 1) / (kTreeWaves * nspan);
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

template <class E, int D, int NT>
__global__ __launch_bounds__(256, D == 128 ? 1 : 2) void tree_attn_kernel(TreeAttnParams p) {
  using V8 = typename E::v8;
  using TL = Tile<D>;
  constexpr int KT = D / 16, DT = D / 32, TILE = kTreeKeys * TL::RB;
  constexpr int COPIES = 2 * TILE / 1024;  // of a K and a V tile
  constexpr int C4 = D / 4;                // 16-byte chunks of an fp32 row
  __shared__ __attribute__((aligned(1024))) char smem[kTreeWaves][2][2][TILE];  // then the waves' o [32 NT][D] fp32
  __shared__ float wm[kTreeWaves][32 * NT], wl[kTreeWaves][32 * NT];
  static_assert(sizeof(smem[0]) >= 32 * NT * D * 4, "a wave's o fits its tiles");
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the row blocks of one (sequence, KV head, span) on one XCD (index mod 8), one after the other
  const int slot = blockIdx.x % (8 * p.blocks), g = blockIdx.x / (8 * p.blocks) * 8 + slot % 8, rb = slot / 8;
  if (g >= p.B * p.Hkv * p.nspan) return;
  const int s = g % p.nspan, pair = g / p.nspan, kvh = pair % p.Hkv, b = pair / p.Hkv;
  const int L = p.t.cached(b), N = p.t.N, RN = p.R * N;
  const TreeTiles tl(L, N, p.nspan);
  if (s * kTreeWaves * tl.per >= tl.all) return;  // the combine does not read this span
  const int t0 = (s * kTreeWaves + wave) * tl.per, t1 = min(tl.all, t0 + tl.per);

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

  // the rows' queries (B operands) and what they see of the tree
  const uint64_t anc = tree_ancestors(p.t, b, lane);
  V8 qop[NT][KT];
  uint64_t seen[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = (rb * NT + nt) * 32 + l32, rc = min(row, RN - 1), node = rc % N;
    const uint16_t* qr = p.q + b * p.sq[0] + (int64_t)(kvh * p.R + rc / N) * p.sq[1] + (int64_t)node * p.sq[2] + 8 * hh;
    const uint64_t a = shfl64(anc, node);
    seen[nt] = row < RN ? a : 0ull;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(qr + 16 * kk);
      qop[nt][kk] = __builtin_bit_cast(V8, seen[nt] ? x : zero4());
    }
  }
  const uint64_t padding = ~__ballot(anc != 0ull);  // nodes whose keys and values are not read

  f32x16 oacc[DT][NT];
  float mrun[NT], lrun[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    mrun[nt] = kTreeNone;
    lrun[nt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) zero16(oacc[dt][nt]);
  }
  const int rbase = TL::row_base(lane);
  const TrBase tbase = TL::tr_base(lane);
  const float c2 = p.scale_log2;

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
      for (int i = lane; i < kTreeKeys * TL::NC; i += 64)
        if (padding >> (n0 + i / TL::NC) & 1) *reinterpret_cast<u32x4*>(vl + i * 16) = zero4();
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    f32x16 st[NT];
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      const V8 a = TL::template row_op<E>(kl, rbase, 0, kk);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) st[nt] = E::mfma(a, qop[nt][kk], kk == 0 ? f32x16{} : st[nt]);
    }
    if (n0 >= 0 || (t + 1) * kTreeKeys > L) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = 8 * (i >> 2) + 4 * hh + (i & 3);
          const bool in = n0 >= 0 ? (seen[nt] >> (n0 + key)) & 1 : t * kTreeKeys + key < L;
          st[nt][i] = in ? st[nt][i] : -INFINITY;
        }
    }
    V8 pk[NT][2];
    float qs[NT];
    // P = 2^(S c2 - m) in 16 bits; the sums add the rounded values, the weights that P V uses
    auto ex = [&](int nt) {
      u32x4 w[2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2][i & 3] = pack2<E>(exp2_fast(__builtin_fmaf(st[nt][2 * i], c2, -mrun[nt])),
                                    exp2_fast(__builtin_fmaf(st[nt][2 * i + 1], c2, -mrun[nt])));
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s0 = E::sum2(w[0][i], s0);
        s1 = E::sum2(w[1][i], s1);
      }
      qs[nt] = s0 + s1;
      pk[nt][0] = __builtin_bit_cast(V8, w[0]);
      pk[nt][1] = __builtin_bit_cast(V8, w[1]);
    };
    bool high = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      ex(nt);
      high |= !(qs[nt] <= kSumLimit);
    }
    // a P above 2^kRescaleSlack (or the first keys): that row's m is raised to its maximum.  Other
    // rows of the wave keep theirs, so a row's result does not depend on the rows beside it.
    if (__builtin_amdgcn_ballot_w64(high)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float v = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) v = fmaxf(v, st[nt][i]);
        const bool raise = max_with_partner(qs[nt] <= kSumLimit ? 0.f : 1.f) > 0.f;
        v = max_with_partner(v) * c2;
        const float m = raise ? fmaxf(mrun[nt], v) : mrun[nt], alpha = exp2_fast(mrun[nt] - m);
        mrun[nt] = m;
        lrun[nt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) oacc[dt][nt][i] *= alpha;
        ex(nt);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) lrun[nt] += qs[nt];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const V8 a = TL::template tr_op<E>(vl, tbase, k2, dt);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) oacc[dt][nt] = E::mfma(a, pk[nt][k2], oacc[dt][nt]);
      }
    if (t + 2 < t1) {
      reads_done();
      stage(t + 2, buf);
    }
  }
  reads_done();

  // the wave's o, 16-byte chunk c of row r at slot c ^ (r mod C4)
  float* ow = reinterpret_cast<float*>(smem[wave]);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 32 + l32;
    const float l = sum_with_partner(lrun[nt]);
    if (hh == 0) {
      wm[wave][r] = seen[nt] ? mrun[nt] : kTreeNone;
      wl[wave][r] = seen[nt] ? l : 0.f;  // padding: no weight anywhere
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = dt * 8 + 2 * q + hh;
        *reinterpret_cast<f32x4*>(ow + r * D + 4 * (c ^ (r % C4))) =
            f32x4{oacc[dt][nt][4 * q], oacc[dt][nt][4 * q + 1], oacc[dt][nt][4 * q + 2], oacc[dt][nt][4 * q + 3]};
      }
  }
  __syncthreads();
  for (int i = tid; i < 32 * NT * C4; i += 64 * kTreeWaves) {
    const int r = i / C4, c = i % C4, row = rb * NT * 32 + r;
    if (row >= RN) continue;
    float M = wm[0][r], lt = 0.f;
#pragma unroll
    for (int w = 1; w < kTreeWaves; ++w) M = fmaxf(M, wm[w][r]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) {
      const float a = exp2_fast(wm[w][r] - M);
      const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem[w]) + r * D + 4 * (c ^ (r % C4)));
      lt = __builtin_fmaf(a, wl[w][r], lt);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(a, x[e], o[e]);
    }
    if (p.nspan == 1) {
      const float inv = 1.f / lt;
      u32x2 y = {pack2<E>(o[0] * inv, o[1] * inv), pack2<E>(o[2] * inv, o[3] * inv)};
      if (lt == 0.f) y = u32x2{0u, 0u};
      *reinterpret_cast<u32x2*>(p.out + (((int64_t)b * p.Hkv + kvh) * RN + row) * D + 4 * c) = y;
    } else {
      float* dst = p.part + (((int64_t)pair * RN + row) * p.nspan + s) * (D + 4);
      *reinterpret_cast<f32x4*>(dst + 4 * c) = o;
      if (c == 0) *reinterpret_cast<f32x2*>(dst + D) = f32x2{M, lt};
    }
  }
}

// Joins the spans of each query row: M = max m_s, o = sum_s 2^(m_s - M) o_s over the
// same sum of l_s.  One thread per 4 values of a row, 8 spans in flight.
template <class E, int D>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeAttnParams p) {
  constexpr int C4 = D / 4, ROW = D + 4, BATCH = 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / C4;
  const int c = i % C4, RN = p.R * p.t.N;
  if (row >= (int64_t)p.B * p.Hkv * RN) return;
  const int b = int(row / ((int64_t)p.Hkv * RN));
  const TreeTiles tl(p.t.cached(b), p.t.N, p.nspan);
  const int ns = (tl.all + kTreeWaves * tl.per - 1) / (kTreeWaves * tl.per);  // spans that held keys
  const float* src = p.part + row * p.nspan * ROW;
  float M = kTreeNone, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < ns; s0 += BATCH) {
    f32x2 ml[BATCH];
    f32x4 x[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const float* r = src + (int64_t)min(s0 + j, ns - 1) * ROW;
      ml[j] = *reinterpret_cast<const f32x2*>(r + D);
      x[j] = *reinterpret_cast<const f32x4*>(r + 4 * c);
    }
    float mn = M;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) mn = fmaxf(mn, ml[j][0]);
    const float a = exp2_fast(M - mn);
    l *= a;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (s0 + j >= ns) continue;
      const float w = exp2_fast(ml[j][0] - mn);
      l = __builtin_fmaf(w, ml[j][1], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, x[j][e], o[e]);
    }
    M = mn;
  }
  const float inv = 1.f / l;
  u32x2 y = {pack2<E>(o[0] * inv, o[1] * inv), pack2<E>(o[2] * inv, o[3] * inv)};
  if (l == 0.f) y = u32x2{0u, 0u};
  *reinterpret_cast<u32x2*>(p.out + row * D + 4 * c) = y;
}

// ===========================================================================
// Accepted nodes into the caches: cache[b, h, cached(b) + j] = node[b, h, path[b, j]]
// for j < count[b], keys and values of up to kCommitLayers layers in one launch.  One thread
// per W 16-bit values; slots j >= count end at once, j the slowest index.
// ===========================================================================
constexpr int kCommitLayers = 32;

struct TreeCommitParams {
  const uint16_t* src[2][kCommitLayers];  // [B, Hkv, N, D]: keys, values
  uint16_t* dst[2][kCommitLayers];        // [B, Hkv, capacity, D]
  int64_t ss[2][3], sd[2][3];             // strides (b, h, n | t), one for all layers
  const int *path, *count;                // [B, N], [B]
  TreeShape t;                            // parents unused
  int layers, Hkv, D;
  int blocks;  // workgroups of a sequence
};

template <int W>
__global__ __launch_bounds__(256) void tree_commit_kernel(TreeCommitParams p) {
  const int b = blockIdx.x / p.blocks, nc = p.D / W;
  int64_t i = (int64_t)(blockIdx.x % p.blocks) * 256 + threadIdx.x;
  const int c = int(i % nc);
  i /= nc;
  const int h = int(i % p.Hkv);
  i /= p.Hkv;
  const int w = int(i % 2);
  i /= 2;
  const int layer = int(i % p.layers);
  const int j = int(i / p.layers);
  if (j >= min(p.count[b], p.t.N)) return;
  const int node = p.path[(int64_t)b * p.t.N + j], pos = p.t.cached(b) + j;
  if (node < 0 || node >= p.t.N || pos >= p.t.capacity) return;
  const uint16_t* s = p.src[w][layer] + b * p.ss[w][0] + (int64_t)h * p.ss[w][1] + (int64_t)node * p.ss[w][2] + W * c;
  uint16_t* d = p.dst[w][layer] + b * p.sd[w][0] + (int64_t)h * p.sd[w][1] + (int64_t)pos * p.sd[w][2] + W * c;
  if constexpr (W == 8) *reinterpret_cast<u32x4*>(d) = *reinterpret_cast<const u32x4*>(s);
  else *d = *s;
}

}  // namespace mt
