// augur_rope_axes.cu — rotary positions with several axes (time, height,
// width), fused with the append of keys and values to the paged pool.
//
// A token has one position per axis; frequency j (0 <= j < head_dim / 2) turns
// with the position of its axis:
//   angle_j = float(position[axis_j]) * inv_freq_j
//   x'[j]          = x[j] cos(angle_j)          - x[j + D/2] sin(angle_j)
//   x'[j + D/2]    = x[j + D/2] cos(angle_j)    + x[j] sin(angle_j)
// for q and k, in float32 and rounded once to the cache dtype; k and v go to
// the token's slot of the pool, q to q_out. (One axis gives the ordinary
// rotation, without the reference's rounding after each of its three tensor
// operations, which rope_scatter_kernel keeps.)
//
// Bound by HBM: every row is read and written once, 2 (heads + 2 kv heads)
// head_dim elements a token. A CTA takes a few tokens: it computes their
// head_dim / 2 angles once for all heads (sin and cos in shared memory: no
// table of positions, so none to grow or to read), with its first pieces of q,
// k and v already on their way, and then turns pieces of 16 bytes of a row's
// first half together with the matching 16 bytes of the second.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "augur_kv.h"
#include "common.cuh"

namespace augur_kv_axes {

using augur_kv_dev::record_status;

struct AxesArgs {
  const char* q;
  char* q_out;
  const char* k;
  const char* v;
  int64_t q_stride[2], q_out_stride[2], k_stride[2], v_stride[2];  // bytes: token, head
  char* k_pool;
  char* v_pool;
  int64_t pool_stride[3];  // bytes: block, head, row
  int64_t num_slots;
  int32_t block_size;
  const int64_t* slots;
  int64_t slot_stride;
  const int64_t* positions;
  int64_t pos_stride[2];  // elements: axis, token
  const float* inv_freq;
  const int32_t* axis;
  int32_t n_axes, hq, hkv, half;
  int32_t pieces;        // of a row's half
  int32_t token_pieces;  // (hq + 2 hkv) * pieces
  int32_t tokens_per_cta;
  int64_t n_tokens;
  int32_t* status;
};

constexpr int kThreads = 256;

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
  T v[VEC];
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(AxesArgs a) {
  extern __shared__ float2 turn[];  // [token of the CTA][frequency]: cos, sin
  using V = Vec<T, VEC>;
  const int64_t t0 = int64_t(blockIdx.x) * a.tokens_per_cta;
  const int n = int(min(int64_t(a.tokens_per_cta), a.n_tokens - t0));
  const int work = n * a.token_pieces;
  const int64_t half_bytes = int64_t(a.half) * int64_t(sizeof(T));

  struct Task {
    const char* src;
    char* dst;  // null: nothing to write
    int t, c;   // the CTA's token; first frequency, or -1 for a v row
  };
  auto task = [&](int p) -> Task {
    Task w;
    w.t = p / a.token_pieces;
    const int r = p - w.t * a.token_pieces;
    int h = r / a.pieces;
    const int c = r - h * a.pieces;
    const int64_t token = t0 + w.t, off = int64_t(c) * int64_t(sizeof(V));
    w.c = c * VEC;
    if (h < a.hq) {
      w.src = a.q + token * a.q_stride[0] + int64_t(h) * a.q_stride[1] + off;
      w.dst = a.q_out + token * a.q_out_stride[0] + int64_t(h) * a.q_out_stride[1] + off;
      return w;
    }
    h -= a.hq;
    const bool is_v = h >= a.hkv;
    if (is_v) {
      h -= a.hkv;
      w.c = -1;
    }
    w.src = is_v ? a.v + token * a.v_stride[0] + int64_t(h) * a.v_stride[1] + off
                 : a.k + token * a.k_stride[0] + int64_t(h) * a.k_stride[1] + off;
    const int64_t slot = __ldg(a.slots + token * a.slot_stride);
    w.dst = nullptr;
    if (slot >= a.num_slots) {
      record_status(a.status, AUGUR_KV_EBOUNDS);
    } else if (slot >= 0) {
      const int64_t block = slot / a.block_size;
      w.dst = (is_v ? a.v_pool : a.k_pool) + block * a.pool_stride[0] + int64_t(h) * a.pool_stride[1] +
              (slot - block * a.block_size) * a.pool_stride[2] + off;
    }
    return w;
  };
  auto load = [&](const Task& w, V& x, V& y) {
    x = *reinterpret_cast<const V*>(w.src);
    y = *reinterpret_cast<const V*>(w.src + half_bytes);
  };
  auto finish = [&](const Task& w, V& x, V& y) {
    if (w.dst == nullptr) return;
    if (w.c >= 0) {
      const float2* cs = turn + w.t * a.half + w.c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 f = cs[j];
        const float p = to_f(x.v[j]), q = to_f(y.v[j]);
        x.v[j] = from_f<T>(p * f.x - q * f.y);
        y.v[j] = from_f<T>(q * f.x + p * f.y);
      }
    }
    *reinterpret_cast<V*>(w.dst) = x;
    *reinterpret_cast<V*>(w.dst + half_bytes) = y;
  };

  // the first piece is on its way while the angles are computed
  Task w0;
  V x0, y0;
  const bool any = int(threadIdx.x) < work;
  if (any) {
    w0 = task(threadIdx.x);
    load(w0, x0, y0);
  }
  for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
    const int t = i / a.half, j = i - t * a.half;
    const int axis = __ldg(a.axis + j);
    float c = 1.f, s = 0.f;
    if (axis >= 0 && axis < a.n_axes)
      sincosf(__fmul_rn(float(__ldg(a.positions + axis * a.pos_stride[0] + (t0 + t) * a.pos_stride[1])),
                        __ldg(a.inv_freq + j)), &s, &c);
    else
      record_status(a.status, AUGUR_KV_EBOUNDS);
    turn[i] = make_float2(c, s);
  }
  __syncthreads();
  if (any) finish(w0, x0, y0);
  for (int p = threadIdx.x + kThreads; p < work; p += 2 * kThreads) {
    const bool two = p + kThreads < work;
    Task w1;
    V x1, y1;
    w0 = task(p);
    load(w0, x0, y0);
    if (two) {
      w1 = task(p + kThreads);
      load(w1, x1, y1);
    }
    finish(w0, x0, y0);
    if (two) finish(w1, x1, y1);
  }
}

template <typename T, int VEC>
int launch(AxesArgs a, cudaStream_t st) {
  a.pieces = a.half / VEC;
  a.token_pieces = (a.hq + 2 * a.hkv) * a.pieces;
  // tokens per CTA: as many as leave two resident waves of CTAs, at most 8
  const int64_t want = a.n_tokens / (int64_t(augur_kv_dev::sm_count()) * 16);
  a.tokens_per_cta = int32_t(want < 1 ? 1 : want > 8 ? 8 : want);
  const int64_t grid = (a.n_tokens + a.tokens_per_cta - 1) / a.tokens_per_cta;
  if (grid > 0x7fffffff) return augur_kv_dev::fail(AUGUR_KV_EINVAL, "rope_axes_scatter: too many tokens");
  rope_axes_kernel<T, VEC><<<unsigned(grid), kThreads, size_t(a.tokens_per_cta) * size_t(a.half) * sizeof(float2), st>>>(a);
  return augur_kv_dev::check_launch("rope_axes_kernel");
}

}  // namespace augur_kv_axes

#define AUGUR_KV_EXPORT extern "C" __attribute__((visibility("default")))

AUGUR_KV_EXPORT int augur_kv_rope_axes_scatter(const augur_kv_rope_axes_args* p, int32_t layer, const void* q,
                                               const void* k, const void* v, void* q_out, const int64_t* slots,
                                               const int64_t* positions, void* stream) {
  using namespace augur_kv_axes;
  using augur_kv_dev::fail;
  augur_kv_dev::g_last_error[0] = '\0';
  if (p == nullptr) return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: null args");
  if (layer < 0 || layer >= p->n_layers)
    return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: layer %d outside [0, %d)", layer, p->n_layers);
  const int es = augur_kv_dev::elem_size(p->dtype);
  if (es == 0) return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: unknown dtype %d", p->dtype);
  if (p->n_tokens < 0) return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: negative sizes");
  if (p->n_tokens == 0) return AUGUR_KV_OK;
  if (q == nullptr || q_out == nullptr || k == nullptr || v == nullptr || p->k_pool == nullptr ||
      p->v_pool == nullptr || slots == nullptr || positions == nullptr || p->inv_freq == nullptr ||
      p->axis_of_frequency == nullptr)
    return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: null pointer argument");
  if (p->n_q_heads <= 0 || p->n_kv_heads <= 0 || p->n_q_heads > 65536 || p->n_kv_heads > 65536 || p->head_dim <= 0 ||
      p->head_dim % 2 != 0 || p->head_dim > 1024 || p->block_size <= 0 || p->num_blocks <= 0 || p->n_axes <= 0)
    return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: bad sizes (head_dim even and at most 1024)");
  AxesArgs a;
  memset(&a, 0, sizeof(a));
  const int64_t layer_bytes = int64_t(layer) * p->pool_strides[0] * es;
  a.q = static_cast<const char*>(q);
  a.q_out = static_cast<char*>(q_out);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.k_pool = static_cast<char*>(p->k_pool) + layer_bytes;
  a.v_pool = static_cast<char*>(p->v_pool) + layer_bytes;
  uintptr_t bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k) |
                   reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(a.k_pool) |
                   reinterpret_cast<uintptr_t>(a.v_pool) | uintptr_t(p->head_dim / 2 * es);
  for (int i = 0; i < 2; ++i) {
    a.q_stride[i] = p->q_strides[i] * es;
    a.q_out_stride[i] = p->q_out_strides[i] * es;
    a.k_stride[i] = p->k_strides[i] * es;
    a.v_stride[i] = p->v_strides[i] * es;
    a.pos_stride[i] = p->position_strides[i];
    bits |= uintptr_t(a.q_stride[i]) | uintptr_t(a.q_out_stride[i]) | uintptr_t(a.k_stride[i]) | uintptr_t(a.v_stride[i]);
  }
  for (int i = 0; i < 3; ++i) {
    a.pool_stride[i] = p->pool_strides[i + 1] * es;
    bits |= uintptr_t(a.pool_stride[i]);
  }
  if ((bits & uintptr_t(es - 1)) != 0) return fail(AUGUR_KV_EINVAL, "rope_axes_scatter: pointers must be aligned to the type");
  a.num_slots = p->num_blocks * p->block_size;
  a.block_size = p->block_size;
  a.slots = slots;
  a.slot_stride = p->slot_stride;
  a.positions = positions;
  a.inv_freq = p->inv_freq;
  a.axis = p->axis_of_frequency;
  a.n_axes = p->n_axes;
  a.hq = p->n_q_heads;
  a.hkv = p->n_kv_heads;
  a.half = p->head_dim / 2;
  a.n_tokens = p->n_tokens;
  a.status = p->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = (bits & 15u) == 0;  // every piece of 16 bytes is aligned; else one element a piece
  if (p->dtype == AUGUR_KV_F32) return wide ? launch<float, 4>(a, st) : launch<float, 1>(a, st);
  if (p->dtype == AUGUR_KV_F16) return wide ? launch<__half, 8>(a, st) : launch<__half, 1>(a, st);
  return wide ? launch<__nv_bfloat16, 8>(a, st) : launch<__nv_bfloat16, 1>(a, st);
}
