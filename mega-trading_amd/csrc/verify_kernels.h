// Verification of a tree of drafted tokens (mt_topk_verify), for gfx950.
//
// The walk starts at node 0, the last token already accepted.  At node u the
// target distribution p is the softmax over the logits of u that are at least
// their k-th largest (as in mt_topk_sample).  u's children are tried in index
// order, child c with token x and the caller's uniform number r:
//   accept (and walk on from c) if r q(x) < p(x),
//   else p becomes max(p - q, 0), scaled to sum 1, and the next child is tried,
// with q the drafter's distribution at u (softmax over its k largest logits) or,
// without drafter logits, all of its weight at x: then p loses x.  Where that
// leaves nothing, by rounding, p stays.  When no child is left the token drawn is
// the first index of the largest p / E, E Exponential(1) noise.  Children drawn
// from q, or chosen without q, thus leave the target's distribution unchanged.
// NaN and -inf logits count as the lowest float, +inf as the highest.
//
// Two launches.  verify_rows_kernel takes every row that the walk may need, one
// workgroup of 1024 threads a row (held in registers as order-preserving keys,
// EPT a thread): the k-th largest key, the maximum, the sum of the kept
// exponentials, and, where they are few, the kept values themselves as a list.
// verify_walk_kernel then walks, one workgroup a sequence: an acceptance needs
// four scalars and none of the vocabulary, a rejection or the draw goes over
// the node's list (a row without one, for k > 1024, k = vocab or many ties, is
// read again).
#pragma once

#include "sample_kernels.h"
#include "tree_kernels.h"

namespace mt {

// What the walk needs of a row: the smallest kept key, the largest logit, the
// sum of exp(x - max) over the kept, and the entries of its list (0: none).
struct RowTop {
  uint32_t kth;
  float max, sum;
  int listed;
};

struct VerifyParams {
  const void* rows[2];  // the target's and the drafter's logits [B, N, V] (the latter null without one)
  int64_t s[2][2];      // strides (b, n), unit last stride
  const int64_t* tokens;   // [B, N]
  const int* parents;      // [N], int64 stride between sequences
  int64_t parents_stride;
  const float* uniform;    // [B, N]
  const float* noise;      // [B, V], row stride ldn
  int64_t ldn;
  RowTop* top;             // workspace [2 or 1][B, N]
  u32x2* list;             // workspace [B, N][kSampleCand]: (key, index) of the target rows
  int* path;               // [B, N]
  int* count;              // [B]
  int64_t* token;          // [B]
  int B, N, V, k;
};

template <int DT>
__device__ __forceinline__ float load_logit(const void* base, int64_t i) {
  return fminf(fmaxf(ops::IO<DT>::load1(base, i), -__FLT_MAX__), __FLT_MAX__);
}

// A node's parent, or -2 for padding: only earlier nodes have children.
__device__ __forceinline__ int verify_parent(const VerifyParams& p, int b, int n) {
  const int up = p.parents[b * p.parents_stride + n];
  return up < n ? up : -2;
}

struct RowLds {
  uint32_t bound[2][kSampleWaves];
  float top[kSampleWaves], buf[kSampleWaves];
  int count[kSampleWaves];
  uint32_t kth;
  __attribute__((aligned(16))) uint32_t key[kSampleCand];
  int idx[kSampleCand];
};

// key: of value tid + 1024 j of the row at slot j, 0 past its end.  A row with a
// list has it in s.key / s.idx on return, behind a barrier.
template <int EPT>
__device__ __forceinline__ RowTop row_top(const uint32_t (&key)[EPT], int V, int k, RowLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t mx = key[0];
#pragma unroll
  for (int j = 1; j < EPT; ++j) mx = max(mx, key[j]);
  // bounds below the k-th key: the smallest over the waves of their ceil(k / 16)-th lane
  // maxima, the largest of their k-th ones (0 where a wave holds fewer values)
  const bool list = k <= kSampleWaveK && k < V;
  uint32_t t1 = 0u, t2 = 0u;
  if (list) {
    const int k1 = (k + kSampleWaves - 1) / kSampleWaves;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c1 = t1 | (1u << bit), c2 = t2 | (1u << bit);
      if (__popcll(__ballot(mx >= c1)) >= k1) t1 = c1;
      if (__popcll(__ballot(mx >= c2)) >= k) t2 = c2;
    }
  }
  const float wmax = wave_reduce<0, true>(mx ? sample_unkey(mx) : -INFINITY);
  if (lane == 0) {
    s.bound[0][wave] = t1;
    s.bound[1][wave] = t2;
    s.top[wave] = wmax;
  }
  if (tid == 0) s.kth = 0xffffffffu;
  __syncthreads();
  RowTop r{0u, s.top[0], 0.f, 0};
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    r.max = fmaxf(r.max, s.top[w]);
    t1 = min(t1, s.bound[0][w]);
    t2 = max(t2, s.bound[1][w]);
  }
  if (list) {
    const uint32_t t = max(max(t1, t2), 1u);  // a key of 0 is no value
    int mine = 0;
#pragma unroll
    for (int j = 0; j < EPT; ++j) mine += __popcll(__ballot(key[j] >= t));
    if (lane == 0) s.count[wave] = mine;
    __syncthreads();
    int at = 0, n = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
      const int c = s.count[w];
      at += w < wave ? c : 0;
      n += c;
    }
    if (n <= kSampleCand) {
#pragma unroll
      for (int j = 0; j < EPT; ++j) {
        const uint64_t mask = __ballot(key[j] >= t);
        if (key[j] >= t) {
          const int slot = at + __popcll(mask & ((1ull << lane) - 1));
          s.key[slot] = key[j];
          s.idx[slot] = tid + j * kSampleThreads;
        }
        at += __popcll(mask);
      }
      const int pad = n + tid;  // up to three zero keys complete the last group of four
      if (tid < 3 && pad < kSampleCand) s.key[pad] = 0u;
      __syncthreads();
      const uint32_t own = tid < n ? s.key[tid] : 0u;
      if (tid < n) {
        int larger = 0;
        for (int c = 0; c < n; c += 4) {
          const u32x4 q = *reinterpret_cast<const u32x4*>(&s.key[c]);
#pragma unroll
          for (int e = 0; e < 4; ++e) larger += q[e] > own ? 1 : 0;
        }
        if (larger < k) atomicMin(&s.kth, own);
      }
      __syncthreads();
      r.kth = s.kth;
      r.listed = n;
      r.sum = block_reduce<false>(own >= r.kth ? expf(sample_unkey(own) - r.max) : 0.f, s.buf);
      return r;
    }
  }
  if (k < V) {  // the largest t with count(key >= t) >= k, bit by bit
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = r.kth | (1u << bit);
      float c = 0.f;
#pragma unroll
      for (int j = 0; j < EPT; ++j) c += key[j] >= cand ? 1.f : 0.f;
      if (block_reduce<false>(c, s.buf) >= (float)k) r.kth = cand;
    }
  } else {
    r.kth = 1u;
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < EPT; ++j)
    if (key[j] >= r.kth) sum += expf(sample_unkey(key[j]) - r.max);
  r.sum = block_reduce<false>(sum, s.buf);
  return r;
}

// One row a workgroup: blockIdx.x = (drafter?, b, n).
template <int DT, int EPT>
__global__ __launch_bounds__(kSampleThreads) void verify_rows_kernel(VerifyParams p) {
  __shared__ RowLds s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = blockIdx.x >= p.B * p.N, row = blockIdx.x - w * p.B * p.N, b = row / p.N, n = row % p.N;
  // a row that no walk can reach or use: of padding, and a drafter's without children
  if (w) {
    if (!__ballot(lane < p.N && lane > n && verify_parent(p, b, lane < p.N ? lane : 0) == n)) return;
  } else if (verify_parent(p, b, n) < -1) {
    return;
  }
  uint32_t key[EPT];
  const int64_t at = b * p.s[w][0] + n * p.s[w][1];
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    const int i = tid + j * kSampleThreads;
    key[j] = i < p.V ? sample_key(load_logit<DT>(p.rows[w], at + i)) : 0u;
  }
  const RowTop r = row_top<EPT>(key, p.V, p.k, s);
  if (tid == 0) p.top[blockIdx.x] = r;
  if (!w && tid < r.listed) p.list[(int64_t)row * kSampleCand + tid] = u32x2{s.key[tid], (uint32_t)s.idx[tid]};
}

// A walk: LDS copies of what every node's test needs, and the node's rejections.
struct WalkLds {
  RowTop top[2][kTreeNodes];
  int parents[kTreeNodes], path[kTreeNodes];
  int64_t tokens[kTreeNodes];
  float uniform[kTreeNodes];
  float logit[2][kTreeNodes];  // of a node's token in its parent's rows
  float sums[kTreeNodes];      // W of p before each rejection (drafter), else:
  int64_t gone[kTreeNodes];    // the rejected tokens
  float buf[kSampleWaves];
  unsigned long long best[kSampleWaves];
};

template <int DT, bool DRAFT>
__global__ __launch_bounds__(kSampleThreads) void verify_walk_kernel(VerifyParams p) {
  __shared__ WalkLds s;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, N = p.N;
  if (tid < N) {
    const int up = verify_parent(p, b, tid);
    const int64_t x = p.tokens[(int64_t)b * N + tid];
    s.parents[tid] = up;
    s.path[tid] = -1;
    s.tokens[tid] = x;
    s.uniform[tid] = p.uniform[(int64_t)b * N + tid];
    const bool asked = up >= 0 && x >= 0 && x < p.V;
#pragma unroll
    for (int w = 0; w <= (DRAFT ? 1 : 0); ++w) {
      s.top[w][tid] = p.top[(int64_t)w * p.B * N + (int64_t)b * N + tid];
      // a token outside the vocabulary has probability 0
      s.logit[w][tid] = asked ? load_logit<DT>(p.rows[w], b * p.s[w][0] + up * p.s[w][1] + x) : -INFINITY;
    }
  }
  __syncthreads();
  auto kept = [](float x, const RowTop& t) { return x > -INFINITY && sample_key(x) >= t.kth ? expf(x - t.max) : 0.f; };
  int here = s.parents[0] == -1 ? 0 : -1, count = 0;  // node 0 padding: no walk
  int64_t drawn = 0;
  while (here >= 0) {
    if (tid == 0) s.path[count] = here;
    ++count;
    uint64_t kids = __ballot(lane < N && s.parents[lane < N ? lane : 0] == here);
    const RowTop tp = s.top[0][here], tq = s.top[DRAFT ? 1 : 0][here];
    const int64_t xat = b * p.s[0][0] + here * p.s[0][1], yat = DRAFT ? b * p.s[1][0] + here * p.s[1][1] : 0;
    const u32x2* list = p.list + ((int64_t)b * N + here) * kSampleCand;
    const int n = tp.listed ? tp.listed : p.V;
    float W = tp.sum;
    int gone = 0;  // rejections that changed p
    // the weight of a word (unnormalised, sum W): its kept exponential, after the rejections so far
    auto weight = [&](float w, float q, int64_t word) {
      for (int j = 0; j < gone; ++j)
        w = DRAFT ? fmaxf(w * (1.f / s.sums[j]) - q, 0.f) : word == s.gone[j] ? 0.f : w;
      return w;
    };
    // f(weight, q, word) over the words of this thread
    auto each = [&](auto f) {
      for (int i = tid; i < n; i += kSampleThreads) {
        int word = i;
        float w;
        if (tp.listed) {
          const u32x2 e = list[i];
          word = (int)e[1];
          w = e[0] >= tp.kth ? expf(sample_unkey(e[0]) - tp.max) : 0.f;
        } else {
          w = kept(load_logit<DT>(p.rows[0], xat + i), tp);
        }
        if (!(w > 0.f)) continue;
        float q = 0.f;
        if constexpr (DRAFT)
          if (gone || kids) q = kept(load_logit<DT>(p.rows[1], yat + word), tq) * (1.f / tq.sum);
        f(weight(w, q, word), q, word);
      }
    };
    int next = -1;
    while (kids) {
      const int c = __builtin_ctzll(kids);
      const int64_t x = s.tokens[c];
      const float q = DRAFT ? kept(s.logit[1][c], tq) * (1.f / tq.sum) : 1.f;
      const float px = weight(kept(s.logit[0][c], tp), q, x) * (1.f / W);
      if (s.uniform[c] * q < px) {
        next = c;
        break;
      }
      float sum = 0.f;
      const float inv = 1.f / W;
      each([&](float w, float qw, int word) { sum += DRAFT ? fmaxf(w * inv - qw, 0.f) : word == x ? 0.f : w; });
      sum = block_reduce<false>(sum, s.buf);
      if (sum > 0.f) {
        if (tid == 0) {
          s.sums[gone] = W;
          s.gone[gone] = x;
        }
        ++gone;
        W = sum;
        __syncthreads();
      }
      kids &= kids - 1;
    }
    here = next;
    if (next >= 0) continue;
    const float inv = 1.f / W;
    const float* noise = p.noise + b * p.ldn;
    unsigned long long best = 0ull;
    each([&](float w, float, int word) {
      const float v = w * inv / noise[word];
      // the larger value, then the lower index
      const unsigned long long y = ((unsigned long long)__float_as_uint(v) << 32) | (0xffffffffu - (uint32_t)word);
      if (w > 0.f && v >= 0.f && y > best) best = y;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor(best, o, 64);
      best = other > best ? other : best;
    }
    if (lane == 0) s.best[tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kSampleWaves; ++v) best = s.best[v] > best ? s.best[v] : best;
    if (best) drawn = (int64_t)(0xffffffffu - (uint32_t)best);
  }
  __syncthreads();
  if (tid < N) p.path[(int64_t)b * N + tid] = s.path[tid];
  if (tid == 0) {
    p.count[b] = count;
    p.token[b] = drawn;
  }
}

}  // namespace mt
