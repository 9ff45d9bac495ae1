// C ABI of generation over drafted trees and of distillation: argument checks,
// launch geometry and dispatch to tree_kernels.h, verify_kernels.h and
// distill_kernels.h.  Declared in include/mt_attention.h and include/mt_ops.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/mt_attention.h"
#include "../../include/mt_ops.h"
#include "distill_kernels.h"
#include "mt_abi.h"
#include "tree_kernels.h"
#include "verify_kernels.h"

namespace {

using mt_abi::device_cus;
using mt_abi::fail;
using mt_abi::ok;
using mt::ops::kDtBF16;
using mt::ops::kDtFP16;
using mt::ops::kDtFP32;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ok() : fail((int)e, "%s launch failed: %s", what, hipGetErrorString(e));
}

int check_type(int dtype, bool fp32) {
  if (dtype == MT_DTYPE_BF16 || dtype == MT_DTYPE_FP16 || (fp32 && dtype == MT_DTYPE_FP32)) return MT_OK;
  return fail(MT_E_DTYPE, "dtype code %d unsupported", dtype);
}

// (b, h, row) strides of a [B, H, rows, D] tensor with unit last stride and 16-byte rows
int check_rows16(const char* name, const void* p, const int64_t* s) {
  if (!p) return fail(MT_E_NULL, "%s is NULL", name);
  if (!aligned16(p)) return fail(MT_E_STRIDE, "%s must be 16-byte aligned", name);
  if (s[3] != 1) return fail(MT_E_STRIDE, "%s: last-dim stride must be 1 (got %lld)", name, (long long)s[3]);
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8)
      return fail(MT_E_STRIDE, "%s: stride %d (%lld) must be a non-negative multiple of 8 elements", name, i,
                  (long long)s[i]);
  // the copies keep 16 rows of offsets in 32-bit registers
  if (s[2] > (int64_t(1) << 24)) return fail(MT_E_STRIDE, "%s: row stride %lld too large", name, (long long)s[2]);
  return MT_OK;
}

int check_tree(int B, int N, const int* parents, int64_t parents_stride, const int* length_dev, int length_stride,
               int length, int capacity) {
  if (B < 1 || N < 1 || N > mt::kTreeNodes)
    return fail(MT_E_SHAPE, "B must be >= 1 and the nodes in [1, %d] (got %d, %d)", mt::kTreeNodes, B, N);
  if (capacity < 0 || capacity > 0x7fffff00)  // tiles past the end are counted in 32 bits
    return fail(MT_E_SHAPE, "capacity %d is negative or too large", capacity);
  if (!parents) return fail(MT_E_NULL, "parents is NULL");
  if (parents_stride != 0 && parents_stride < N)
    return fail(MT_E_STRIDE, "parents stride %lld must be 0 or at least the nodes", (long long)parents_stride);
  if (length_dev && (length_stride < 0 || length_stride > 1))
    return fail(MT_E_STRIDE, "length stride %d must be 0 or 1", length_stride);
  if (!length_dev && (length < 0 || length > capacity))
    return fail(MT_E_SHAPE, "length %d outside [0, capacity %d]", length, capacity);
  return MT_OK;
}

int check_heads(int Hq, int Hkv) {
  if (Hq < 1 || Hkv < 1 || Hq % Hkv)
    return fail(MT_E_SHAPE, "query heads (%d) must equal key/value heads (%d) multiplied by repeats", Hq, Hkv);
  return MT_OK;
}

mt::TreeShape shape(const int* parents, int64_t parents_stride, const int* length_dev, int length_stride, int length,
                    int capacity, int N) {
  mt::TreeShape t{};
  t.parents = parents;
  t.parents_stride = parents_stride;
  t.length_dev = length_dev;
  t.length_stride = length_stride;
  t.length = length;
  t.capacity = capacity;
  t.N = N;
  return t;
}

// The attention's launch: row waves of a workgroup (RW, 0 for the few-row kernel), row blocks of a KV
// head and workgroups its keys are split over.
struct Split {
  int rw, blocks, keys, groups;
  int64_t nspan;
};
Split split(int64_t B, int64_t Hkv, int64_t R, int N, int64_t cached, int D) {
  Split s{};
  const int64_t rows = R * N, cus = device_cus(), tiles32 = (cached + 31) / 32 + (N + 31) / 32;
  // The smallest row blocks that still give no CU two workgroups (a workgroup fills a CU): more CUs work, and a
  // workgroup's tiles go to more key groups.  But every block reads all keys, which counts when there are many of
  // them: up to 96 tiles of 32 keys a CU for blocks of 32 rows (32 at D = 128), 4 times that for blocks of
  // twice the rows.  us at blocks of 32 / 64 / 128 / 256 rows, span joins included; KV heads of all sequences, rows
  // of each, D, keys:
  //    64,  64,  64,   545:  8.4 / 12.3                    16, 256,  64, 10000:  31.3 / 26.3 / 28.4 / 37.9
  //    64, 128,  64,  1000: 11.5 / 14.8 / 20.5             64, 256,  64,  1000:  21.8 / 16.2 / 23.8 / 29.8
  //   128, 256,  64,  3000: 73.0 / 48.6 / 41.9 / 53.4     256, 256,  64, 10000:   377 /  286 /  259 /  231
  //    16, 128, 128,  1000: 15.4 / 15.9 / 19.6             64, 128, 128,  3000:  36.9 / 31.0 / 33.7
  //    64, 128, 128, 10000:  105 / 82.6 / 71.3             64, 256, 128,   300:  22.9 / 12.7 / 26.0 / 35.1
  int64_t most_tiles = (D == 128 ? 32 : 96) * cus;
  int take = 32;
  for (;; take *= 2, most_tiles *= 4) {
    s.blocks = (int)((rows + take - 1) / take);
    const int64_t n = B * Hkv * s.blocks;
    if (s.blocks == 1 || take == 256 || (n <= cus && n * tiles32 <= most_tiles)) break;
  }
  const int waves = D == 128 ? 8 : 16;
  s.rw = take == 32 ? 0 : take / 32;
  s.keys = s.rw ? 16 * s.rw : mt::kTreeKeys;
  s.groups = s.rw ? waves / s.rw : waves / 2;
  const int64_t tiles = (cached + s.keys - 1) / s.keys + (N + s.keys - 1) / s.keys;
  // Up to 192 keys a key group stay with one workgroup: joining spans is another launch (one span against
  // several, 8 heads over 2 KV heads of 64: 5 nodes on 200 of 1024 keys 6.1 / 10.2 us; 32 sequences of 16 nodes on 545
  // of 1024 keys 8.5 / 11.9, on 1500 keys 11.8 / 12.8).  More are split over all CUs, down to two tiles.
  const int64_t want = cus / std::max<int64_t>(1, B * Hkv * s.blocks);
  const int64_t most = tiles * s.keys <= 192 * s.groups ? 1 : (tiles + 2 * s.groups - 1) / (2 * s.groups);
  s.nspan = std::max<int64_t>(1, std::min(want, most));
  return s;
}

template <class E, int D>
void launch_tree(const mt::TreeAttnParams& p, int rw, unsigned grid, hipStream_t st) {
  const dim3 few(64 * mt::tree_few_waves<D>()), many(64 * mt::tree_waves<D>());
  if (rw == 0) hipLaunchKernelGGL((mt::tree_attn_kernel<E, D>), dim3(grid), few, 0, st, p);
  else if (rw == 2) hipLaunchKernelGGL((mt::tree_attn_rows_kernel<E, D, 2>), dim3(grid), many, 0, st, p);
  else if (rw == 4) hipLaunchKernelGGL((mt::tree_attn_rows_kernel<E, D, 4>), dim3(grid), many, 0, st, p);
  else hipLaunchKernelGGL((mt::tree_attn_rows_kernel<E, D, 8>), dim3(grid), many, 0, st, p);
  if (p.nspan == 1) return;
  // up to 8 spans come in one batch of loads, and threads that share a row would only add their meeting
  // (2 spans, 12288 rows of 128: 6.8 / 17.5 us; 118 spans, 512 rows of 64: 10.3 / 4.5)
  const int64_t n = (int64_t)p.B * p.Hkv * p.R * p.t.N, few_rows = 256 / (D / 4), many_rows = few_rows / 8;
  if (p.nspan <= 8)
    hipLaunchKernelGGL((mt::tree_combine_kernel<E, D, 1>), dim3((unsigned)((n + few_rows - 1) / few_rows)), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((mt::tree_combine_kernel<E, D, 8>), dim3((unsigned)((n + many_rows - 1) / many_rows)), dim3(256), 0,
                       st, p);
}

// Nodes of a sequence whose rows are taken before the walk, in rows a CU.  A drafter's tokens are mostly
// accepted and its walks long, and each node that is taken on the way costs two rows one after the other; a walk
// without a drafter's probabilities is short.  Rows and walk, us, at 1, 2 and 4 rows a CU; fp32:
//   drafter, 32 sequences of 16 nodes, 16384 words:  6 + 25,  8 + 21, 15 + 10;  32001 words: 10 + 75, 20 + 51, 36 + 12
//   drafter, 16 sequences of 64 nodes, 16384 words:  6 + 48,  8 + 50, 16 + 12;  32001 words: 10 + 39, 20 + 39, 37 + 16
//   none, 16 sequences of 64 nodes, 16384 words:     6 + 12,  8 + 9,  16 + 9
//   none, 64 sequences of 64 nodes, 32001 16-bit words: 9.5 + 15, 13 + 15, 22 + 15
int verify_ahead(int64_t B, int N, int vocab, bool draft) {
  const int64_t rows = (draft ? 4 : vocab <= 16384 ? 2 : 1) * (int64_t)device_cus();
  return (int)std::max<int64_t>(1, std::min<int64_t>(N, rows / (B * (draft ? 2 : 1))));
}

// Workspace of the verification: the rows' RowTop, then the target rows' lists.
size_t verify_tops(int64_t B, int ahead, bool draft) {
  return ((size_t)B * ahead * (draft ? 2 : 1) * sizeof(mt::RowTop) + 255) / 256 * 256;
}

template <int DT, int T, int C>
void launch_verify(const mt::VerifyParams& p, hipStream_t st) {
  const dim3 rows((unsigned)((int64_t)p.B * p.ahead * (p.rows[1] ? 2 : 1))), block(T), walks((unsigned)p.B);
  hipLaunchKernelGGL((mt::verify_rows_kernel<DT, T, C>), rows, block, 0, st, p);
  if (p.rows[1]) hipLaunchKernelGGL((mt::verify_walk_kernel<DT, T, C, true>), walks, block, 0, st, p);
  else hipLaunchKernelGGL((mt::verify_walk_kernel<DT, T, C, false>), walks, block, 0, st, p);
}

// A row in 32 registers a thread, 64 for fp32 (a quarter for a short vocabulary): 64 values.  Twice the threads and
// half the values take longer (rows and walk, 16384 fp32 words: 15.2 + 10.0 us against 17.8 + 10.0; 32001 fp32
// words 10.7 + 15.7 against 12.7 + 19.1, 16-bit words 9.5 + 14.8 against 11.8 + 17.9): what a wave does for itself, the
// ballots of the bound above all, is much of a row's time.
template <int DT>
void launch_verify_v(const mt::VerifyParams& p, hipStream_t st) {
  if (p.V <= 4096) launch_verify<DT, 256, 2>(p, st);
  else if (p.V <= 16384) launch_verify<DT, 256, 8>(p, st);
  else launch_verify<DT, 512, 8>(p, st);
}

int check_distill(int64_t ld, int64_t rows, int vocab, int entries, float temperature, int dtype) {
  int rc;
  if ((rc = check_type(dtype, true))) return rc;
  if (rows < 0 || rows > 0x7fffffffLL) return fail(MT_E_SHAPE, "rows must be in [0, 2^31) (got %lld)", (long long)rows);
  if (vocab < 1) return fail(MT_E_SHAPE, "vocab %d unsupported (positive)", vocab);
  if (entries < 1 || entries > mt::kDistillEntries)
    return fail(MT_E_SHAPE, "entries of a row must be in [1, %d] (got %d)", mt::kDistillEntries, entries);
  if (!(temperature > 0.f) || !(1.f / temperature > 0.f) || !(temperature < INFINITY) || !(1.f / temperature < INFINITY))
    return fail(MT_E_SHAPE, "temperature must be positive and finite (got %g)", (double)temperature);
  if (ld < vocab) return fail(MT_E_STRIDE, "row stride %lld must be >= vocab", (long long)ld);
  return MT_OK;
}

int check_type_aligned(const char* name, const void* p, int dtype) {
  if (!p) return fail(MT_E_NULL, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % (dtype == MT_DTYPE_FP32 ? 4 : 2))
    return fail(MT_E_STRIDE, "%s must be aligned to its type", name);
  return MT_OK;
}

}  // namespace

extern "C" {

int mt_tree_rope(const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, const float* rope_cos,
                 const float* rope_sin, int table_rows, const int* parents, int64_t parents_stride,
                 const int* length_dev, int length_stride, int length, int B, int Hq, int Hkv, int N, int D, int dtype,
                 void* stream) {
  int rc;
  if ((rc = check_type(dtype, true)) || (rc = check_heads(Hq, Hkv))) return rc;
  if (D < 8 || D % 8 || D > 1024) return fail(MT_E_SHAPE, "head size %d unsupported (a multiple of 8 up to 1024)", D);
  if (table_rows < 1) return fail(MT_E_ROPE, "RoPE tables have no rows");
  if ((rc = check_tree(B, N, parents, parents_stride, length_dev, length_stride, length, table_rows))) return rc;
  if (!strides || !rope_cos || !rope_sin || !q_out || !k_out)
    return fail(MT_E_NULL, "strides, the RoPE tables and the outputs must be non-NULL");
  if ((rc = check_rows16("q", q, strides)) || (rc = check_rows16("k", k, strides + 4))) return rc;
  if (!aligned16(rope_cos) || !aligned16(rope_sin) || !aligned16(q_out) || !aligned16(k_out))
    return fail(MT_E_STRIDE, "the RoPE tables and the outputs must be 16-byte aligned");
  mt::TreeRopeParams p{};
  p.src[0] = q;
  p.src[1] = k;
  p.dst[0] = q_out;
  p.dst[1] = k_out;
  for (int i = 0; i < 3; ++i) {
    p.s[0][i] = strides[i];
    p.s[1][i] = strides[4 + i];
  }
  p.heads[0] = Hq;
  p.heads[1] = Hkv;
  p.t = shape(parents, parents_stride, length_dev, length_stride, length, table_rows, N);
  p.cos = rope_cos;
  p.sin = rope_sin;
  p.table_rows = table_rows;
  p.D = D;
  const int64_t chunks = ((int64_t)Hq + Hkv) * N * (D / 8), blocks = (chunks + 255) / 256;
  if (blocks * B > 0x7fffffffLL || chunks > 0x7fffffffLL) return fail(MT_E_SHAPE, "too many values");
  p.blocks = (int)blocks;
  const dim3 grid((unsigned)(blocks * B));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MT_DTYPE_BF16) hipLaunchKernelGGL((mt::tree_rope_kernel<kDtBF16>), grid, dim3(256), 0, st, p);
  else if (dtype == MT_DTYPE_FP16) hipLaunchKernelGGL((mt::tree_rope_kernel<kDtFP16>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((mt::tree_rope_kernel<kDtFP32>), grid, dim3(256), 0, st, p);
  return launched("tree RoPE");
}

size_t mt_tree_attn_workspace_size(int B, int Hq, int Hkv, int N, int keys, int D) {
  if (B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || N < 1 || keys < 0 || D < 1) return 0;
  const Split s = split(B, Hkv, Hq / Hkv, N, keys, D);
  if (s.nspan == 1) return 0;
  return ((size_t)B * Hq * N * (size_t)s.nspan * (size_t)(D + 4) * sizeof(float) + 255) / 256 * 256;
}

int mt_tree_attn(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache, void* o,
                 const int64_t* strides, const int* parents, int64_t parents_stride, const int* length_dev,
                 int length_stride, int length, int capacity, int B, int Hq, int Hkv, int N, int D, float scale,
                 int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_type(dtype, false)) || (rc = check_heads(Hq, Hkv)) ||
      (rc = check_tree(B, N, parents, parents_stride, length_dev, length_stride, length, capacity)))
    return rc;
  if (D != 32 && D != 64 && D != 128) return fail(MT_E_SHAPE, "head size %d unsupported (32, 64 or 128)", D);
  if (!(scale > 0.f)) return fail(MT_E_SHAPE, "scale must be positive (got %g)", (double)scale);
  if (!strides) return fail(MT_E_NULL, "strides is NULL");
  if ((rc = check_rows16("q", q, strides)) || (rc = check_rows16("k", k, strides + 4)) ||
      (rc = check_rows16("v", v, strides + 8)))
    return rc;
  if (capacity > 0 && ((rc = check_rows16("k_cache", k_cache, strides + 12)) ||
                       (rc = check_rows16("v_cache", v_cache, strides + 16))))
    return rc;
  if (!o || !aligned16(o)) return fail(o ? MT_E_STRIDE : MT_E_NULL, "o must be non-NULL and 16-byte aligned");
  const int keys = length_dev ? capacity : length;
  const Split s = split(B, Hkv, Hq / Hkv, N, keys, D);
  const size_t need = mt_tree_attn_workspace_size(B, Hq, Hkv, N, keys, D);
  if (need && (!workspace || !aligned16(workspace)))
    return fail(workspace ? MT_E_STRIDE : MT_E_NULL, "workspace must be non-NULL and 16-byte aligned");
  if (workspace_bytes < need)
    return fail(MT_E_WORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
  mt::TreeAttnParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.kc = static_cast<const uint16_t*>(k_cache);
  p.vc = static_cast<const uint16_t*>(v_cache);
  p.out = static_cast<uint16_t*>(o);
  p.part = static_cast<float*>(workspace);
  for (int i = 0; i < 3; ++i) {
    p.sq[i] = strides[i];
    p.sk[i] = strides[4 + i];
    p.sv[i] = strides[8 + i];
    p.skc[i] = strides[12 + i];
    p.svc[i] = strides[16 + i];
  }
  p.t = shape(parents, parents_stride, length_dev, length_stride, length, capacity, N);
  p.B = B;
  p.Hkv = Hkv;
  p.R = Hq / Hkv;
  p.nspan = (int)s.nspan;
  p.blocks = s.blocks;
  p.keys = s.keys;
  p.groups = s.groups;
  p.scale_log2 = scale * mt::kLog2e;
  const int64_t groups = ((int64_t)B * Hkv * s.nspan + 7) / 8 * 8;
  const int64_t rows = (int64_t)B * Hq * N;
  if (groups * s.blocks > 0x7fffffffLL || rows > 0x7fffffffLL)
    return fail(MT_E_SHAPE, "too many query rows (%lld)", (long long)rows);
  const unsigned grid = (unsigned)(groups * s.blocks);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MT_DTYPE_BF16) {
    if (D == 32) launch_tree<mt::BF16, 32>(p, s.rw, grid, st);
    else if (D == 64) launch_tree<mt::BF16, 64>(p, s.rw, grid, st);
    else launch_tree<mt::BF16, 128>(p, s.rw, grid, st);
  } else {
    if (D == 32) launch_tree<mt::FP16, 32>(p, s.rw, grid, st);
    else if (D == 64) launch_tree<mt::FP16, 64>(p, s.rw, grid, st);
    else launch_tree<mt::FP16, 128>(p, s.rw, grid, st);
  }
  return launched("tree attention");
}

int mt_tree_commit(const void* const* keys, const void* const* values, void* const* key_caches,
                   void* const* value_caches, int layers, const int64_t* strides, const int* path, const int* count,
                   const int* length_dev, int length_stride, int length, int capacity, int B, int Hkv, int N, int D,
                   int dtype, void* stream) {
  int rc;
  if ((rc = check_type(dtype, false))) return rc;
  static const int kNoTree = -1;  // check_tree's parents, unused here
  if ((rc = check_tree(B, N, &kNoTree, 0, length_dev, length_stride, length, capacity))) return rc;
  if (Hkv < 1 || D < 1 || layers < 0)
    return fail(MT_E_SHAPE, "Hkv and D must be >= 1 and layers >= 0 (got %d, %d, %d)", Hkv, D, layers);
  if (layers == 0 || capacity == 0) return ok();
  if (!keys || !values || !key_caches || !value_caches || !strides || !path || !count)
    return fail(MT_E_NULL, "keys, values, the caches, strides, path and count must be non-NULL");
  bool wide = D % 8 == 0;
  for (int i = 0; i < 4; ++i) {
    if (strides[4 * i + 3] != 1) return fail(MT_E_STRIDE, "every last-dim stride must be 1");
    for (int j = 0; j < 3; ++j) wide = wide && strides[4 * i + j] % 8 == 0;
  }
  for (int l = 0; l < layers; ++l) {
    const void* ptr[4] = {keys[l], values[l], key_caches[l], value_caches[l]};
    for (const void* x : ptr) {
      if (!x) return fail(MT_E_NULL, "layer %d: keys, values and the caches must be non-NULL", l);
      if (reinterpret_cast<uintptr_t>(x) % 2) return fail(MT_E_STRIDE, "layer %d: misaligned pointer", l);
      wide = wide && aligned16(x);
    }
  }
  mt::TreeCommitParams p{};
  for (int j = 0; j < 3; ++j) {
    p.ss[0][j] = strides[j];
    p.ss[1][j] = strides[4 + j];
    p.sd[0][j] = strides[8 + j];
    p.sd[1][j] = strides[12 + j];
  }
  p.path = path;
  p.count = count;
  p.t = shape(nullptr, 0, length_dev, length_stride, length, capacity, N);
  p.Hkv = Hkv;
  p.D = D;
  hipStream_t st = (hipStream_t)stream;
  for (int l0 = 0; l0 < layers; l0 += mt::kCommitLayers) {
    p.layers = std::min(mt::kCommitLayers, layers - l0);
    for (int l = 0; l < p.layers; ++l) {
      p.src[0][l] = static_cast<const uint16_t*>(keys[l0 + l]);
      p.src[1][l] = static_cast<const uint16_t*>(values[l0 + l]);
      p.dst[0][l] = static_cast<uint16_t*>(key_caches[l0 + l]);
      p.dst[1][l] = static_cast<uint16_t*>(value_caches[l0 + l]);
    }
    // The nodes are shared out while that takes no more than 4 workgroups a CU (8 layers, 4 trees of 64 nodes,
    // 8 heads of 128: 24 us with one thread a node, 13.5 with up to 2 workgroups a CU, 11.3 with 4, 11.5 with 8).
    const int64_t n = (int64_t)p.layers * 2 * Hkv * (wide ? D / 8 : D);
    p.split = (int)std::max<int64_t>(1, std::min<int64_t>(N, 4 * (int64_t)device_cus() * 256 / (n * B)));
    const int64_t blocks = (n * p.split + 255) / 256;
    if (blocks * B > 0x7fffffffLL) return fail(MT_E_SHAPE, "too many values");
    p.blocks = (int)blocks;
    const dim3 grid((unsigned)(blocks * B));
    if (wide) hipLaunchKernelGGL((mt::tree_commit_kernel<8>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((mt::tree_commit_kernel<1>), grid, dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail((int)e, "tree commit launch failed: %s", hipGetErrorString(e));
  }
  return ok();
}

size_t mt_topk_verify_workspace_size(int B, int N, int vocab, int k, int draft) {
  if (B < 1 || N < 1 || N > mt::kTreeNodes || vocab < 1 || k < 1) return 0;
  const int ahead = verify_ahead(B, N, vocab, draft != 0);
  return verify_tops(B, ahead, draft != 0) + (size_t)B * ahead * mt::kVerifyList * sizeof(mt::u32x2);
}

int mt_topk_verify(const void* logits, const void* draft_logits, const int64_t* strides, const int64_t* tokens,
                   const int* parents, int64_t parents_stride, const float* uniform, const float* noise,
                   int64_t noise_row_stride, int* path, int* count, int64_t* token, int B, int N, int vocab, int k,
                   int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_type(dtype, true))) return rc;
  if (B < 0) return fail(MT_E_SHAPE, "B must be >= 0 (got %d)", B);
  if (N < 1 || N > mt::kTreeNodes) return fail(MT_E_SHAPE, "nodes must be in [1, %d] (got %d)", mt::kTreeNodes, N);
  if (vocab < 1 || vocab > 32 * mt::kSampleThreads)
    return fail(MT_E_SHAPE, "vocab must be in [1, %d] (got %d)", 32 * mt::kSampleThreads, vocab);
  if (k < 1 || k > vocab) return fail(MT_E_SHAPE, "k must be in [1, vocab] (got %d)", k);
  if (B == 0) return ok();
  if (!strides || !tokens || !parents || !uniform || !noise || !path || !count || !token)
    return fail(MT_E_NULL, "strides, tokens, parents, uniform, noise, path, count and token must be non-NULL");
  if (parents_stride != 0 && parents_stride < N)
    return fail(MT_E_STRIDE, "parents stride %lld must be 0 or at least the nodes", (long long)parents_stride);
  if ((rc = check_type_aligned("logits", logits, dtype))) return rc;
  if (draft_logits && (rc = check_type_aligned("draft_logits", draft_logits, dtype))) return rc;
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0) return fail(MT_E_STRIDE, "strides must not be negative");
  if (noise_row_stride < vocab && B > 1)
    return fail(MT_E_STRIDE, "noise row stride %lld must be >= vocab", (long long)noise_row_stride);
  if ((int64_t)B * N > 0x3fffffff) return fail(MT_E_SHAPE, "too many nodes (%d x %d)", B, N);
  if (!workspace || !aligned16(workspace))
    return fail(workspace ? MT_E_STRIDE : MT_E_NULL, "workspace must be non-NULL and 16-byte aligned");
  const size_t need = mt_topk_verify_workspace_size(B, N, vocab, k, draft_logits != nullptr);
  if (workspace_bytes < need)
    return fail(MT_E_WORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
  mt::VerifyParams p{};
  p.ahead = verify_ahead(B, N, vocab, draft_logits != nullptr);
  p.rows[0] = logits;
  p.rows[1] = draft_logits;
  for (int i = 0; i < 2; ++i) {
    p.s[0][i] = strides[i];
    p.s[1][i] = strides[2 + i];
  }
  p.tokens = tokens;
  p.parents = parents;
  p.parents_stride = parents_stride;
  p.uniform = uniform;
  p.noise = noise;
  p.ldn = noise_row_stride;
  p.top = static_cast<mt::RowTop*>(workspace);
  p.list = reinterpret_cast<mt::u32x2*>(static_cast<char*>(workspace) + verify_tops(B, p.ahead, draft_logits != nullptr));
  p.path = path;
  p.count = count;
  p.token = token;
  p.B = B;
  p.N = N;
  p.V = vocab;
  p.k = k;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MT_DTYPE_BF16) launch_verify_v<kDtBF16>(p, st);
  else if (dtype == MT_DTYPE_FP16) launch_verify_v<kDtFP16>(p, st);
  else launch_verify_v<kDtFP32>(p, st);
  return launched("verification");
}

int mt_topk_distill_fwd(const void* logits, int64_t row_stride, const float* teacher, const int64_t* index,
                        int64_t rows, int vocab, int entries, float temperature, float* row_state, float* loss,
                        int dtype, void* stream) {
  int rc;
  if ((rc = check_distill(row_stride, rows, vocab, entries, temperature, dtype))) return rc;
  if (!loss || !row_state) return fail(MT_E_NULL, "loss and row_state must be non-NULL");
  if (!aligned16(row_state)) return fail(MT_E_STRIDE, "row_state must be 16-byte aligned");
  if (rows > 0) {
    if ((rc = check_type_aligned("logits", logits, dtype))) return rc;
    if (!teacher || !index) return fail(MT_E_NULL, "teacher and index must be non-NULL");
  }
  mt::DistillParams p{};
  p.x = logits;
  p.ldx = row_stride;
  p.teacher = teacher;
  p.index = index;
  p.V = vocab;
  p.K = entries;
  p.rows = rows;
  p.inv_t = 1.f / temperature;
  p.row = row_state;
  hipStream_t st = (hipStream_t)stream;
  if (rows > 0) {
    const dim3 grid((unsigned)rows);
    if (dtype == MT_DTYPE_BF16) hipLaunchKernelGGL((mt::distill_fwd_kernel<kDtBF16>), grid, dim3(256), 0, st, p);
    else if (dtype == MT_DTYPE_FP16) hipLaunchKernelGGL((mt::distill_fwd_kernel<kDtFP16>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((mt::distill_fwd_kernel<kDtFP32>), grid, dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail((int)e, "distillation launch failed: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(mt::distill_sum_kernel, dim3(1), dim3(1024), 0, st, row_state, rows, temperature * temperature,
                     loss);
  return launched("distillation");
}

int mt_topk_distill_bwd(const void* logits, int64_t row_stride, const float* teacher, const int64_t* index,
                        const float* row_state, const float* grad, void* dlogits, int64_t rows, int vocab, int entries,
                        float temperature, int dtype, void* stream) {
  int rc;
  if ((rc = check_distill(row_stride, rows, vocab, entries, temperature, dtype))) return rc;
  if (rows == 0) return ok();
  if ((rc = check_type_aligned("logits", logits, dtype)) || (rc = check_type_aligned("dlogits", dlogits, dtype))) return rc;
  if (!teacher || !index || !row_state || !grad)
    return fail(MT_E_NULL, "teacher, index, row_state and grad must be non-NULL");
  if (!aligned16(row_state)) return fail(MT_E_STRIDE, "row_state must be 16-byte aligned");
  mt::DistillParams p{};
  p.x = logits;
  p.ldx = row_stride;
  p.teacher = teacher;
  p.index = index;
  p.V = vocab;
  p.K = entries;
  p.rows = rows;
  p.inv_t = 1.f / temperature;
  p.row = const_cast<float*>(row_state);
  p.grad = grad;
  p.dx = dlogits;
  const dim3 grid((unsigned)rows);
  hipStream_t st = (hipStream_t)stream;
  // A gradient larger than the 256 MB cache in front of the memory cannot stay there: stored past it, it
  // leaves the logits (32768 x 16384 bf16: 355 us, and 221 for the forward of the next step; 354 + 198 past it).
  const bool past = rows * vocab * (dtype == MT_DTYPE_FP32 ? 4 : 2) > int64_t(256) << 20;
  const bool few = entries <= mt::kDistillFew;
#define MT_DISTILL_BWD2(DT, PAST)                                                                                  \
  if (few) hipLaunchKernelGGL((mt::distill_bwd_kernel<DT, PAST, mt::kDistillFew>), grid, dim3(256), 0, st, p);     \
  else hipLaunchKernelGGL((mt::distill_bwd_kernel<DT, PAST, mt::kDistillEntries>), grid, dim3(256), 0, st, p)
#define MT_DISTILL_BWD(DT)                 \
  if (past) { MT_DISTILL_BWD2(DT, true); } \
  else { MT_DISTILL_BWD2(DT, false); }
  if (dtype == MT_DTYPE_BF16) { MT_DISTILL_BWD(kDtBF16) }
  else if (dtype == MT_DTYPE_FP16) { MT_DISTILL_BWD(kDtFP16) }
  else { MT_DISTILL_BWD(kDtFP32) }
#undef MT_DISTILL_BWD2
#undef MT_DISTILL_BWD
  return launched("distillation");
}

}  // extern "C"
