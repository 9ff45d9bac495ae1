// Distillation from a teacher's top logits, forward and backward, for gfx950.
//
// Row r has K entries (index i_j, teacher logit y_j); an index below 0 or a logit of
// -inf is no entry, and a row without entries counts nothing.  With the temperature T,
//   p = softmax(y / T) over the entries,  log q = log softmax(x / T) over the vocabulary,
//   loss = T^2 / n sum_r sum_j p_j (log p_j - log q[i_j]),  n = rows with entries,
//   dx = g T / n (q - P),  P[v] = sum of the p_j with i_j = v.
// Entries of one index each have their own term.  An index past the vocabulary makes
// the row NaN.
//
// Bound by memory: the forward reads each logit once (a running maximum and sum), the
// backward reads it and writes its gradient once.  One workgroup of 256 threads a row,
// 8 values a load, kDistillAhead loads of a thread in flight; rows need no alignment
// beyond their type's (an odd vocabulary), since a global load of 16 bytes takes any
// address.  The backward starts with the rows that the forward read last: part of them
// is still in the 256 MB cache in front of the memory (688 -> 670 us for the step).
//
// 32768 rows of 16384 bf16 logits, 64 entries: forward 178 to 198 us (5.4 to 6.0 TB/s), its
// sum 11, backward 354 to 373 (5.8 to 6.1 TB/s read and written).
#pragma once

#include "storage.h"

namespace mt {

constexpr int kDistillEntries = 1024;  // of a row
constexpr int kDistillAhead = 4;       // loads of a thread in flight

struct DistillParams {
  const void* x;  // [rows, V], row stride ldx
  int64_t ldx;
  const float* teacher;  // [rows, K]
  const int64_t* index;  // [rows, K]
  int V, K;
  int64_t rows;
  float inv_t;
  // [rows + 1, 4]: the row's sum of p (log p - log q), the largest logit M, the sum of exp((x - M) / T)
  // (two numbers where one, the logarithm, would lose bits with the logits' size), 1 (0 without entries);
  // then n
  float* row;
  // backward
  const float* grad;  // incoming gradient
  void* dx;           // [rows, V] contiguous
};

template <bool MAX>
__device__ __forceinline__ float block_reduce_256(float v, float* buf) {
  v = wave_reduce<0, MAX>(v);
  __syncthreads();  // the previous reduction's reads are done
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return red_op<MAX>(red_op<MAX>(buf[0], buf[1]), red_op<MAX>(buf[2], buf[3]));
}

constexpr int kDistillPer = kDistillEntries / 256;  // entries of a thread

template <int PER>
struct Entries {
  int64_t idx[PER];  // -1 where there is no entry
  float p[PER], logp[PER];
  bool any;
};

// The row's entries and their probabilities, entry threadIdx.x + 256 j at slot j.
template <int PER>
__device__ __forceinline__ Entries<PER> load_entries(const DistillParams& a, int64_t row, float* buf) {
  Entries<PER> e;
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = threadIdx.x + 256 * j;
    e.idx[j] = -1;
    e.logp[j] = -INFINITY;
    if (i < a.K) {
      e.idx[j] = a.index[row * a.K + i];
      if (e.idx[j] >= 0) e.logp[j] = a.teacher[row * a.K + i] * a.inv_t;
      if (e.logp[j] == -INFINITY) e.idx[j] = -1;
    }
    m = fmaxf(m, e.logp[j]);
  }
  m = block_reduce_256<true>(m, buf);
  // NaN logits: fmaxf passes over them, the sum does not
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    e.p[j] = e.idx[j] < 0 ? 0.f : expf(e.logp[j] - m);
    sum += e.p[j];
  }
  sum = block_reduce_256<false>(sum, buf);
  e.any = !(sum == 0.f);
  const float inv = 1.f / sum, off = m + logf(sum);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    e.p[j] = e.idx[j] < 0 ? 0.f : e.p[j] * inv;  // also where a NaN among the entries makes inv one
    e.logp[j] -= off;
  }
  return e;
}

template <int DT>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillParams a) {
  constexpr int PER = kDistillPer;
  __shared__ float buf[4];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t base = row * a.ldx;
  const Entries<PER> e = load_entries<PER>(a, row, buf);
  if (!e.any) {
    if (tid == 0) *reinterpret_cast<f32x4*>(a.row + 4 * row) = f32x4{0.f, 0.f, 1.f, 0.f};
    return;
  }
  // a running maximum m and sum of 2^(x c - m c), c = log2(e) / T
  const float c2 = a.inv_t * kLog2e;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float mx, float (&v)[8]) {
    if (mx > m) {
      s *= exp2_fast((m - mx) * c2);
      m = mx;
    }
    const float from = m == -INFINITY ? 0.f : m;  // before any number: -inf adds 0, NaN stays NaN
#pragma unroll
    for (int j = 0; j < 8; ++j) s += exp2_fast((v[j] - from) * c2);
  };
  const int nvec = a.V / 8;
  for (int c0 = tid; c0 < nvec; c0 += 256 * kDistillAhead) {
    typename ops::IO<DT>::Raw r[kDistillAhead];
#pragma unroll
    for (int i = 0; i < kDistillAhead; ++i) r[i] = ops::load8_any<DT>(a.x, base + 8 * min(c0 + 256 * i, nvec - 1));
#pragma unroll
    for (int i = 0; i < kDistillAhead; ++i) {
      if (c0 + 256 * i >= nvec) continue;
      float v[8];
      ops::IO<DT>::unpack(r[i], v);
      float mx = v[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, v[j]);
      add(mx, v);
    }
  }
  if (tid < a.V - 8 * nvec) {
    float v[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
    v[0] = ops::IO<DT>::load1(a.x, base + 8 * nvec + tid);
    add(v[0], v);
  }
  const float M = block_reduce_256<true>(m, buf);
  s = block_reduce_256<false>(m == -INFINITY ? s : s * exp2_fast((m - M) * c2), buf);
  const float logs = logf(s);
  float loss = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (e.idx[j] >= 0 && e.p[j] != 0.f) {
      const bool in = e.idx[j] < a.V;
      const float xi = ops::IO<DT>::load1(a.x, base + (in ? e.idx[j] : 0));
      loss += in ? e.p[j] * (e.logp[j] - ((xi - M) * a.inv_t - logs)) : __builtin_nanf("");
    }
  loss = block_reduce_256<false>(loss, buf);
  if (tid == 0) *reinterpret_cast<f32x4*>(a.row + 4 * row) = f32x4{loss, M, s, 1.f};
}

// loss = T^2 sum / n and n, in a fixed order and 64 bits: one workgroup.
__global__ __launch_bounds__(1024) void distill_sum_kernel(float* row, int64_t rows, float t2, float* loss) {
  __shared__ double part[2][16];
  double s = 0., n = 0.;
  for (int64_t i = threadIdx.x; i < rows; i += 16 * 1024) {
    f32x4 v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = *reinterpret_cast<const f32x4*>(row + 4 * min(i + 1024 * j, rows - 1));
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (i + 1024 * j < rows) {
        s += v[j][0];
        n += v[j][3];
      }
  }
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = s;
    part[1][threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = n = 0.;
    for (int w = 0; w < 16; ++w) {
      s += part[0][w];
      n += part[1][w];
    }
    *loss = n > 0. ? (float)(s * t2 / n) : 0.f;
    row[4 * rows] = (float)n;
  }
}

// A gradient is stored once, whole: a column that an entry names takes its P on the way.  So the entries
// are laid out first: those of one index share the sum of their p, in their order, and the first of them goes into
// a table by the column's group of 8.  A bitmap of hashed indexes tells which could have another (a few in a hundred at
// 1024 entries), and a wave looks for each of those (8192 rows of 16384 bf16 logits: 84 us with 64 entries, where every
// thread looking through all of them for its own takes 93; 102 with 1024, 1099 so).  Stored again after the others
// instead, the named columns cost 65 of 425 us at 32768 rows with 64 entries: parts of lines that had left the caches.
//
// Up to kDistillFew entries have a smaller table: less LDS to clear, and more rows on a CU (28337 rows of 663 fp32
// logits, 6 entries: 54 us, 84 in the large one; 32768 rows of 16384 bf16 logits, 64 entries: 372 and 367).
constexpr int kDistillFew = 64;

template <int ENT, int TABLE>
struct DistillLds {
  float buf[4];
  uint32_t table[TABLE];      // the first entry of a group's, plus 1
  int idx[ENT];               // -1: none
  float prob[ENT], sum[ENT];  // p, and of all entries of the index
  uint16_t next[ENT];         // entry of the group, plus 1
  uint16_t list[ENT];         // entries that could have another
  int count;
};

// PAST: the gradient goes past the caches.
template <int DT, bool PAST, int ENT>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillParams a) {
  constexpr int TABLE = ENT == kDistillFew ? 256 : 2048, BITS = TABLE / 2 * 32;  // both bitmaps lie where the table will be
  constexpr int PER = ENT > 256 ? ENT / 256 : 1;  // entries of a thread
  __shared__ DistillLds<ENT, TABLE> lds;
  const int64_t row = a.rows - 1 - blockIdx.x;  // the rows that the forward read last first: some are still in a cache
  const int tid = threadIdx.x;
  const int64_t base = row * a.ldx, out = row * a.V;
  const int nvec = a.V / 8;
  const f32x4 r = *reinterpret_cast<const f32x4*>(a.row + 4 * row);
  if (r[3] == 0.f) {
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = tid; c < nvec; c += 256) ops::store8_any<DT, PAST>(a.dx, out + 8 * c, z);
    if (tid < a.V - 8 * nvec) ops::IO<DT>::store1(a.dx, out + 8 * nvec + tid, 0.f);
    return;
  }
  const Entries<PER> e = load_entries<PER>(a, row, lds.buf);
  bool bad = false;
  int idx[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + 256 * j;
    idx[j] = e.idx[j] < a.V ? (int)e.idx[j] : -1;
    if (i < ENT) {
      lds.idx[i] = idx[j];
      lds.prob[i] = lds.sum[i] = e.p[j];
    }
    bad |= e.p[j] != 0.f && e.idx[j] >= a.V;
  }
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < TABLE / 256; ++i) lds.table[tid + 256 * i] = 0u;
  };
  clear();
  if (tid == 0) lds.count = 0;
  const float c2 = a.inv_t * kLog2e, M = r[1], inv = 1.f / r[2];
  float scale = *a.grad / (a.row[4 * a.rows] * a.inv_t);
  if (__syncthreads_or(bad)) scale = __builtin_nanf("");
  const float qs = inv * scale;
  auto insert = [&](int i, int v) { lds.next[i] = (uint16_t)atomicExch(&lds.table[v / 8 % TABLE], (uint32_t)i + 1u); };
  uint32_t *seen = lds.table, *twice = lds.table + BITS / 32;
  auto bit = [](int v) { return (uint32_t)v * 2654435761u >> (ENT == kDistillFew ? 20 : 17); };
  static_assert(BITS == (ENT == kDistillFew ? 1 << 12 : 1 << 15), "the hash's bits");
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (idx[j] < 0) continue;
    const uint32_t h = bit(idx[j]), one = 1u << (h & 31);
    if (atomicOr(&seen[h >> 5], one) & one) atomicOr(&twice[h >> 5], one);
  }
  __syncthreads();
  bool alone[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t h = bit(idx[j]);
    alone[j] = idx[j] >= 0 && !(twice[h >> 5] >> (h & 31) & 1u);
    if (idx[j] >= 0 && !alone[j]) lds.list[atomicAdd(&lds.count, 1)] = (uint16_t)(tid + 256 * j);
  }
  __syncthreads();
  clear();
  const int n = lds.count, lane = tid & 63;
  for (int k = tid >> 6; k < n; k += 4) {  // in any order: an entry's sum is over all of them in theirs
    const int at = lds.list[k], v = lds.idx[at];
    float P = 0.f;
    bool later = false;  // one of the index comes before
    for (int i = lane; i < a.K; i += 64) {
      const bool same = lds.idx[i] == v;
      P += same ? lds.prob[i] : 0.f;
      later |= same && i < at;
    }
    P = wave_reduce<0, false>(P);
    const bool any = __ballot(later) != 0;
    if (lane == 0) {
      lds.sum[at] = P;
      lds.next[at] = any;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (idx[j] >= 0 && (alone[j] || !lds.next[tid + 256 * j])) insert(tid + 256 * j, idx[j]);
  __syncthreads();
  for (int c0 = tid; c0 < nvec; c0 += 256 * kDistillAhead) {
    typename ops::IO<DT>::Raw r[kDistillAhead];
#pragma unroll
    for (int i = 0; i < kDistillAhead; ++i) r[i] = ops::load8_any<DT>(a.x, base + 8 * min(c0 + 256 * i, nvec - 1));
#pragma unroll
    for (int i = 0; i < kDistillAhead; ++i) {
      const int c = c0 + 256 * i;
      if (c >= nvec) continue;
      float v[8];
      ops::IO<DT>::unpack(r[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = exp2_fast((v[j] - M) * c2) * qs;
      for (uint32_t h = lds.table[c % TABLE]; h; h = lds.next[h - 1]) {
        const int at = lds.idx[h - 1];
        if (at / 8 != c) continue;
        const float P = lds.sum[h - 1] * scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] -= at % 8 == j ? P : 0.f;
      }
      ops::store8_any<DT, PAST>(a.dx, out + 8 * c, v);
    }
  }
  if (tid < a.V - 8 * nvec) {
    const int i = 8 * nvec + tid;
    float v = exp2_fast((ops::IO<DT>::load1(a.x, base + i) - M) * c2) * qs;
    for (uint32_t h = lds.table[nvec % TABLE]; h; h = lds.next[h - 1])
      if (lds.idx[h - 1] == i) v -= lds.sum[h - 1] * scale;
    ops::IO<DT>::store1(a.dx, out + i, v);
  }
}

}  // namespace mt
