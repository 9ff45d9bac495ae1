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
// Two launches.  verify_rows_kernel takes rows that the walk may need, one workgroup
// a row: the k-th largest logit, the maximum, the sum of the kept exponentials, and,
// where they are few, the kept values themselves as a list.  verify_walk_kernel then
// walks, one workgroup a sequence: an acceptance needs four scalars and none of the
// vocabulary, a rejection or the draw goes over the node's list (a row without one,
// for large k or many ties, is read again).
//
// A walk visits a few nodes, but which is known only as it goes.  The rows of the
// first `ahead` nodes of every sequence are taken before it, all at once: as many as
// the card holds at a time.  A node past them is taken when the walk reaches it.
//
// Bound by latency: one row alone takes 7 to 8 us from its loads over the bound, the list and the ranks to
// the sum, a node of the walk 1 to 3 us.  32 sequences of 16 nodes with a drafter, 16384 fp32 words:
// 15.5 us for the 67 MB of 1024 rows (4.3 TB/s) and 10.0 for the walks; 64 sequences of 64 nodes without one,
// 32001 bf16 words: 9.4 us for the 16 MB of 256 rows and 13.8 for the walks.  Without a list the walk goes over
// whole rows: every word kept, 21 sequences of 46 nodes without a drafter, 21338 words: 9.9 and 32 us (a
// rejected word's weight is subtracted; passes over the row instead took 111); 16 of 32 nodes with one, 32000 words:
// 27 and 104; k = 2000 there: 78 (the k-th largest by bits) and 145.
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
  RowTop* top;             // workspace [2 or 1][B, ahead]
  u32x2* list;             // workspace [B, ahead][kVerifyList]: (key, index) of the target rows
  int* path;               // [B, N]
  int* count;              // [B]
  int64_t* token;          // [B]
  int B, N, V, k, ahead;
};

constexpr int kVerifyList = 1024;  // values of a list

// A logit as the operator counts it: finite, and no negative zero (its key is another).
__device__ __forceinline__ float as_logit(float x) { return fminf(fmaxf(x, -__FLT_MAX__), __FLT_MAX__) + 0.f; }
template <int DT>
__device__ __forceinline__ float load_logit(const void* base, int64_t i) {
  return as_logit(ops::IO<DT>::load1(base, i));
}

// A node's parent, or -2 for padding: only earlier nodes have children.
__device__ __forceinline__ int verify_parent(const VerifyParams& p, int b, int n) {
  const int up = p.parents[b * p.parents_stride + n];
  return up < n ? up : -2;
}

template <int T>
struct RowLds {
  __attribute__((aligned(16))) uint32_t key[kVerifyList];
  int idx[kVerifyList];
  float buf[T / 64], top[T / 64];
  uint32_t bound[2][T / 64];
  int count[T / 64];
  uint32_t kth;
};

// x of the wave's lanes up to this one, added
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, rows of 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// block-wide max or sum; barriers at both ends of buf's use
template <int T, bool MAX>
__device__ __forceinline__ float reduce_all(float v, float* buf) {
  v = wave_reduce<0, MAX>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = buf[0];
#pragma unroll
  for (int w = 1; w < T / 64; ++w) r = red_op<MAX>(r, buf[w]);
  return r;
}

// A row in registers as it was loaded: slot 8 c + e of a thread holds value word(c, V) + e, 8
// consecutive values a load.  The loads need no branch: the one that would reach past the row's end, and
// those behind it, take the last 8 values instead.  What is no value, or one of a slot before, is NaN:
// every comparison and maximum passes over it.
template <int DT, int T, int C>
struct Row {
  typename ops::IO<DT>::Raw r[C];

  static __device__ __forceinline__ int word(int c, int V) {
    return min(8 * ((int)threadIdx.x + T * c), max(V - 8, 0));
  }
  __device__ __forceinline__ void load(const void* base, int64_t at, int V) {
    const float none = __builtin_nanf("");
    if (V < 8) {  // shorter than a load: the first thread's first slots
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = threadIdx.x == 0 && e < V ? ops::IO<DT>::load1(base, at + e) : none;
      put(0, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = none;
#pragma unroll
      for (int c = 1; c < C; ++c) put(c, v);
      return;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) r[c] = ops::load8_any<DT>(base, at + word(c, V));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int first = 8 * ((int)threadIdx.x + T * c) - word(c, V);
      if (first > 0) {
        float v[8];
        ops::IO<DT>::unpack(r[c], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e >= first ? v[e] : none;
        put(c, v);
      }
    }
  }
  // the 8 values of a load.  Each pass unpacks for itself: kept from pass to pass the values would take
  // twice the registers of the row.
  __device__ __forceinline__ void get(int c, float (&v)[8]) const {
    typename ops::IO<DT>::Raw y = r[c];
    asm volatile("" : "+v"(y.w[0]));
    if constexpr (DT == ops::kDtFP32) asm volatile("" : "+v"(y.w[1]));
    ops::IO<DT>::unpack(y, v);
  }
  // f(value, slot) over the slots
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float v[8];
      get(c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) f(v[e], 8 * c + e);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

 private:
  __device__ __forceinline__ void put(int c, const float* v) {
    if constexpr (DT == ops::kDtFP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[c].w[e / 4][e % 4] = __float_as_uint(v[e]);
    } else {
      using E = typename std::conditional<DT == ops::kDtBF16, BF16, FP16>::type;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[c].w[0][e] = pack2<E>(v[2 * e], v[2 * e + 1]);  // exact
    }
  }
};

// The key of the k-th largest value, as a bound: the largest t with count(key >= t) >= k in the bits that keys of
// the type differ in (the lowest 16 of a bf16 value's are alike, 13 of an fp16 value's).  Keys below -inf's
// are those of NaN, which nothing exceeds: where the k-th largest is -inf, t is 0.
template <int DT, int T, int C>
__device__ __forceinline__ uint32_t kth_key(const Row<DT, T, C>& x, int k, float* buf) {
  constexpr int LAST = DT == ops::kDtBF16 ? 16 : DT == ops::kDtFP16 ? 13 : 0;
  uint32_t t = 0u;
  for (int bit = 31; bit >= LAST; --bit) {
    const uint32_t cand = t | (1u << bit);
    const float c = sample_unkey(cand);
    int n = 0;
    x.each([&](float v, int) { n += v >= c ? 1 : 0; });
    if (reduce_all<T, false>((float)n, buf) >= (float)k) t = cand;
  }
  return t;
}

// A row's RowTop, the same on every thread; one with a list has it in s.key / s.idx
// (ordered by thread and slot), behind a barrier.
//
// The values that count are those >= t, t below the k-th largest and at least max - 110, where
// an exponential is 0.  k <= T: every wave finds the ceil(k / waves)-th and the k-th
// largest of its lanes' maxima, a ballot a bit; at least k values are >= the smallest
// of the former and >= the largest of the latter.  Two to four times k random values pass;
// in LDS, a value that fewer than k of them exceed is kept: ties of the k-th stay.  k > T:
// the k-th largest itself, bit by bit with block-wide counts.
template <int DT, int T, int C>
__device__ __forceinline__ RowTop row_top(const void* base, int64_t row, int V, int k, RowLds<T>& s) {
  constexpr int W = T / 64;
  Row<DT, T, C> x;
  x.load(base, row, V);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float m = -INFINITY;
  x.each([&](float v, int) { m = fmaxf(m, v); });
  uint32_t t1 = 0u, t2 = 0u;
  if (k <= T && k < V) {
    const uint32_t mx = sample_key(m + 0.f);
    const int k1 = (k + W - 1) / W;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c1 = t1 | (1u << bit), c2 = t2 | (1u << bit);
      if (__popcll(__ballot(mx >= c1)) >= k1) t1 = c1;
      if (__popcll(__ballot(mx >= c2)) >= k) t2 = c2;
    }
  }
  const float wmax = wave_reduce<0, true>(m);
  if (lane == 0) {
    s.bound[0][wave] = t1;
    s.bound[1][wave] = t2;
    s.top[wave] = wmax;
  }
  if (tid == 0) s.kth = 0xffffffffu;
  __syncthreads();
  float top = s.top[0];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    top = fmaxf(top, s.top[w]);
    t1 = min(t1, s.bound[0][w]);
    t2 = max(t2, s.bound[1][w]);
  }
  RowTop r{0u, fminf(top, __FLT_MAX__), 0.f, 0};
  if (!(top > -__FLT_MAX__)) {  // nothing above the lowest float: all words alike
    r.max = -__FLT_MAX__;
    r.sum = (float)V;
    return r;
  }
  r.kth = sample_key(r.max - 110.f + 0.f);
  // +inf counts as the highest float, whose words it must not push out
  if (k < V) r.kth = max(r.kth, min(k <= T ? max(t1, t2) : kth_key(x, k, s.buf), sample_key(__FLT_MAX__)));
  const float t = sample_unkey(r.kth);
  uint32_t in[(C + 3) / 4] = {};  // the slots that count, 32 a word, the first in the highest bit
  x.each([&](float v, int j) { in[j / 32] += in[j / 32] + (v >= t ? 1u : 0u); });
  int mine = 0;
#pragma unroll
  for (int w = 0; w < (C + 3) / 4; ++w) mine += __popc(in[w]);
  const int upto = wave_scan(mine);
  if (lane == 63) s.count[wave] = upto;
  __syncthreads();
  int at = upto - mine, n = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int c = s.count[w];
    at += w < wave ? c : 0;
    n += c;
  }
  if (n <= kVerifyList) {
// the indexes from the registers; the values are loaded once more, in a thread of their own each: from
    // the registers, which nothing can index, every one of them would be stored under a condition
#pragma unroll
    for (int w = 0; w < (C + 3) / 4; ++w) {
      constexpr int kSlots = 8 * (C < 4 ? C : 4);
      for (uint32_t bits = in[w]; bits; ++at) {
        const int bit = 31 - __builtin_clz(bits), slot = kSlots - 1 - bit;
        s.idx[at] = Row<DT, T, C>::word(4 * w + slot / 8, V) + slot % 8;
        bits ^= 1u << bit;
      }
    }
    __syncthreads();
    for (int i = tid; i < n; i += T) s.key[i] = sample_key(load_logit<DT>(base, row + s.idx[i]));
    const int pad = n + tid;  // zero keys complete the last group of 64
    if (tid < 63 && pad < kVerifyList) s.key[pad] = 0u;
    __syncthreads();
    if (k < V && k <= T) {
      float least = INFINITY;  // of the values that fewer than k exceed; four threads count for one
      for (int i = tid / 4; i - tid / 4 < n; i += T / 4) {
        const uint32_t own = s.key[min(i, n - 1)];
        int larger = 0;
        for (int c = 4 * (tid & 3); c < n; c += 64) {
          u32x4 q[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) q[g] = *reinterpret_cast<const u32x4*>(&s.key[c + 16 * g]);
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) larger += q[g][e] > own ? 1 : 0;
        }
        larger += __builtin_amdgcn_update_dpp(0, larger, 0xB1, 0xf, 0xf, false);  // the lanes of a quad
        larger += __builtin_amdgcn_update_dpp(0, larger, 0x4E, 0xf, 0xf, false);
        if (larger < k) least = fminf(least, sample_unkey(own));
      }
      least = -wave_reduce<0, true>(-least);
      if (lane == 0 && least < INFINITY) atomicMin(&s.kth, sample_key(least + 0.f));
      __syncthreads();
      r.kth = s.kth;
    }
    float sum = 0.f;  // every wave for itself: the list is short
    for (int i = lane; i < n; i += 64)
      if (s.key[i] >= r.kth) sum += expf(sample_unkey(s.key[i]) - r.max);
    r.sum = wave_reduce<0, false>(sum);
    r.listed = n;
    return r;
  }
  // more values than the list holds: with k <= T the bound may lie below the k-th largest
  if (k < V && k <= T) r.kth = max(r.kth, min(kth_key(x, k, s.buf), sample_key(__FLT_MAX__)));
  const float least = sample_unkey(r.kth);
  float sum = 0.f;
  x.each([&](float v, int) { sum += v >= least ? expf(fminf(v, __FLT_MAX__) - r.max) : 0.f; });
  r.sum = reduce_all<T, false>(sum, s.buf);
  return r;
}

// One row a workgroup: blockIdx.x = (drafter?, b, n) with n < ahead.
template <int DT, int T, int C>
__global__ __launch_bounds__(T) void verify_rows_kernel(VerifyParams p) {
  __shared__ RowLds<T> s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int rows = p.B * p.ahead, w = blockIdx.x >= rows, row = blockIdx.x - w * rows, b = row / p.ahead, n = row % p.ahead;
  // a row that no walk can reach or use: of padding, and a drafter's without children
  if (w) {
    if (!__ballot(lane < p.N && lane > n && verify_parent(p, b, lane < p.N ? lane : 0) == n)) return;
  } else if (verify_parent(p, b, n) < -1) {
    return;
  }
  const RowTop r = row_top<DT, T, C>(p.rows[w], b * p.s[w][0] + n * p.s[w][1], p.V, p.k, s);
  if (tid == 0) p.top[blockIdx.x] = r;
  if (!w)
    for (int i = tid; i < r.listed; i += T) p.list[(int64_t)row * kVerifyList + i] = u32x2{s.key[i], (uint32_t)s.idx[i]};
}

// A walk: LDS copies of what every node's test needs, and the node's rejections.
template <int T>
struct WalkLds {
  RowTop top[2][kTreeNodes];
  int parents[kTreeNodes], path[kTreeNodes];
  int64_t tokens[kTreeNodes];
  float uniform[kTreeNodes];
  float logit[2][kTreeNodes];  // of a node's token in its parent's rows
  float sums[kTreeNodes];      // 1 / sum of p before each rejection,
  int64_t gone[kTreeNodes];    // and the rejected tokens
  float buf[T / 64];
  unsigned long long best[T / 64];
  RowLds<T> row;  // of a node past the rows taken ahead
};

template <int DT, int T, int C, bool DRAFT>
__global__ __launch_bounds__(T) void verify_walk_kernel(VerifyParams p) {
  __shared__ WalkLds<T> s;
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
      if (tid < p.ahead) s.top[w][tid] = p.top[((int64_t)w * p.B + b) * p.ahead + tid];
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
    const int64_t xat = b * p.s[0][0] + here * p.s[0][1], yat = DRAFT ? b * p.s[1][0] + here * p.s[1][1] : 0;
    const bool ready = here < p.ahead;
    RowTop tp, tq{};
    if (__builtin_expect(ready, 1)) {
      tp = s.top[0][here];
      if constexpr (DRAFT) tq = s.top[1][here];
    } else {
      if constexpr (DRAFT)
        if (kids) {
          __syncthreads();  // the last reads of the row's LDS are done
          tq = row_top<DT, T, C>(p.rows[1], yat, p.V, p.k, s.row);
        }
      __syncthreads();
      tp = row_top<DT, T, C>(p.rows[0], xat, p.V, p.k, s.row);
    }
    const u32x2* list = p.list + ((int64_t)b * p.ahead + here) * kVerifyList;
    const int n = tp.listed;
    double W = tp.sum, whole = W;  // p's sum, and the last that a pass over its words gave
    int gone = 0;  // rejections that changed p
    // the weight of a word (unnormalised, sum W): its kept exponential, after the rejections so far
    auto weight = [&](float w, float q, int64_t word) {
      for (int j = 0; j < gone; ++j)
        w = DRAFT ? fmaxf(w * s.sums[j] - q, 0.f) : word == s.gone[j] ? 0.f : w;
      return w;
    };
    // an entry of the node's list: the word, its kept exponential (0: none) and the drafter's probability
    struct Entry {
      int word;
      float w, q;
    };
    const bool asks = kids != 0;
    const float qinv = DRAFT && asks ? 1.f / tq.sum : 0.f;
    auto entry = [&](int i) {
      Entry e{0, 0.f, 0.f};
      if (i >= n) return e;
      const u32x2 x = ready ? list[i] : u32x2{s.row.key[i], (uint32_t)s.row.idx[i]};
      e.word = (int)x[1];
      e.w = x[0] >= tp.kth ? expf(sample_unkey(x[0]) - tp.max) : 0.f;
      if constexpr (DRAFT)
        if (asks && e.w > 0.f) e.q = kept(load_logit<DT>(p.rows[1], yat + e.word), tq) * qinv;
      return e;
    };
    // f(weight, q, word) over the words of this thread.  Its first entry is loaded once a node, when a rejection
    // or the draw first needs it: lists are mostly shorter than the workgroup.  Without a list, 8 words a load.
    Entry own;
    bool loaded = false;
    auto each = [&](auto f) {
      if (n) {
        if (!loaded) own = entry(tid);
        loaded = true;
        if (own.w > 0.f) f(weight(own.w, own.q, own.word), own.q, own.word);
        for (int i = tid + T; i < n; i += T) {
          const Entry e = entry(i);
          if (e.w > 0.f) f(weight(e.w, e.q, e.word), e.q, e.word);
        }
        return;
      }
      for (int i = 8 * tid; i < p.V; i += 8 * T) {
        float x[8], y[8] = {};
        const int m = p.V - i;
        if (m >= 8) {
          const auto xr = ops::load8_any<DT>(p.rows[0], xat + i);
          if constexpr (DRAFT)
            if (asks) ops::IO<DT>::unpack(ops::load8_any<DT>(p.rows[1], yat + i), y);
          ops::IO<DT>::unpack(xr, x);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = e < m ? ops::IO<DT>::load1(p.rows[0], xat + i + e) : -INFINITY;
            if constexpr (DRAFT)
              if (asks && e < m) y[e] = ops::IO<DT>::load1(p.rows[1], yat + i + e);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = e < m ? kept(as_logit(x[e]), tp) : 0.f;
          if (!(w > 0.f)) continue;
          float q = 0.f;
          if constexpr (DRAFT)
            if (asks) q = kept(as_logit(y[e]), tq) * qinv;
          f(weight(w, q, i + e), q, i + e);
        }
      }
    };
    int next = -1;
    while (kids) {
      const int c = __builtin_ctzll(kids);
      const int64_t x = s.tokens[c];
      const float q = DRAFT ? kept(s.logit[1][c], tq) * qinv : 1.f;
      const float inv = 1.f / (float)W, wx = weight(kept(s.logit[0][c], tp), q, x);
      if (s.uniform[c] * q < wx * inv) {
        next = c;
        break;
      }
      double left = W - wx;
      // p loses x alone: its sum less x's weight, while that takes no more than half of what was added up
      if (DRAFT || left < 0.5 * whole) {
        float sum = 0.f;
        each([&](float w, float qw, int word) { sum += DRAFT ? fmaxf(w * inv - qw, 0.f) : word == x ? 0.f : w; });
        left = whole = reduce_all<T, false>(sum, s.buf);
      }
      if (left > 0.) {
        if (tid == 0) {
          s.sums[gone] = inv;
          s.gone[gone] = x;
        }
        ++gone;
        W = left;
        __syncthreads();
      }
      kids &= kids - 1;
    }
    here = next;
    if (next >= 0) continue;
    const float inv = 1.f / (float)W;
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
    for (int v = 0; v < T / 64; ++v) best = s.best[v] > best ? s.best[v] : best;
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
