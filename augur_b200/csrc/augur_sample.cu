// augur_sample.cu — one token per row of logits: temperature, top-k, top-p and
// min-p sampling from a given uniform number.
//
// For a row x with maximum m and temperature T:
//   z_i = (x_i - m) * (1 / T)          (z = 0 where x_i == m)
//   e_i = exp(z_i),  w_i = floor(2^31 e_i)
// The weights are whole numbers, so every sum below is exact in 64 bits and
// the token does not depend on the order in which threads add: the same row
// gives the same token whatever the batch, the cluster size or the path taken.
// (2^-31 of the largest weight is where a weight becomes zero; the sum of
// 2^21 vocabulary entries stays below the 53 bits a double holds exactly.)
//   top-k  the k largest z, ties to the lowest index
//   top-p  of those, in falling order, the entries before which less than
//          ceil(p * their sum) has been passed (the first always stays)
//   min-p  of those, the entries with e_i >= min_p
//   token  the first index, in rising order, at which the kept weights'
//          running sum passes floor(u * their sum)
//
// What bounds it: a row is read once (the floor is its bytes over the HBM
// rate); the rest is the latency of a handful of cluster exchanges.
//  * A row belongs to a cluster of 1 to 8 CTAs; each keeps its part of the row
//    in shared memory as float32, so HBM is read once and the later passes run
//    from shared memory.
//  * Only entries that can still matter get a weight. With top-k, entries
//    below a bound of the k-th largest (the smallest, over the CTAs, of their
//    ceil(k / CTAs)-th largest per-thread maximum: at least k entries reach
//    it) are dropped by one comparison. With top-p alone a coarse histogram
//    of the entries within e^-12 of the maximum shows where the nucleus ends.
//    What remains (at most kList entries, in index order) goes to CTA 0 of the
//    cluster, which sorts it, cuts it and draws.
//  * Where more than kList entries remain (flat rows) the cut is found by a
//    radix search over the bits of |z| (count for top-k, mass for top-p), and
//    the draw walks the row in place; a row with neither top-k nor top-p walks
//    at once.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "augur_kv.h"
#include "common.cuh"

namespace augur_kv_smp {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kList = 2048;     // most entries CTA 0 sorts
constexpr int kBins = 64;       // coarse bins of |z| in [0, kBinRange)
constexpr float kBinRange = 12.f;
constexpr float kBinScale = kBins / kBinRange;
constexpr int kDigits = 256;    // radix search: 8 bits a level
constexpr int kMaxCluster = 8;
constexpr float kNegInf = -INFINITY;
constexpr float kUnit = 2147483648.f;  // 2^31
constexpr uint32_t kDead = 0x7f800000u;  // key of z = -inf

struct SampleArgs {
  const char* logits;
  int64_t row_stride;  // bytes
  int32_t vocab;
  const float* uniform;
  const float* temperature;  // per-row values, or null: the scalar
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s, top_p_s, min_p_s;
  int32_t top_k_s;
  int64_t* tokens;
  float* logprobs;  // may be null
  int32_t granules;  // 16-byte granules a CTA's part holds at most (its shared memory)
};

// What the CTAs of a cluster tell one another (each writes its own copy).
struct Shared {
  float cta_max, cta_tau;
  uint32_t count, ties;
  unsigned long long mass;
  uint32_t warp_count[kWarps];
  unsigned long long warp_mass[kWarps];
  uint32_t hist_count[kDigits];
  unsigned long long hist_mass[kDigits];
  // results of a CTA-wide step, written by one thread
  uint32_t r0, r1;
  unsigned long long r2, r3;
};

template <typename T> struct Logit;
template <> struct Logit<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float one(const char* p) { return *reinterpret_cast<const float*>(p); }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
};
template <> struct Logit<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(const char* p) {
    return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
  }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Logit<__half> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(const char* p) {
    return __half2float(*reinterpret_cast<const __half*>(p));
  }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
};

__device__ __forceinline__ float no_nan(float x) { return x == x ? x : kNegInf; }  // a NaN is never drawn
// floats as unsigned integers of the same order
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// The row's scale: z of an entry, its weight, and its key (bits of |z|: rising
// keys are falling z; kDead for entries that can never be drawn).
struct Scale {
  float m, inv;  // inv = 0: greedy
  bool greedy;
  __device__ __forceinline__ float z(float x) const {
    if (x == m) return 0.f;
    const float v = (x - m) * inv;
    return (greedy || !(v <= 0.f)) ? kNegInf : v;  // -inf * 0 and the like: dead
  }
};
__device__ __forceinline__ uint32_t key_of(float z) { return __float_as_uint(fabsf(z)); }
__device__ __forceinline__ float z_of(uint32_t key) { return -__uint_as_float(key); }
__device__ __forceinline__ uint32_t weight(float e) { return __float2uint_rz(e * kUnit); }

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_scan(V v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

// Whole numbers from a double: ceil(p * s) and floor(u * s), in range.
__device__ __forceinline__ unsigned long long mass_needed(float p, unsigned long long s) {
  const double need = ceil(double(p) * double(s));
  return need >= 1.0 ? (unsigned long long)need : 1ull;
}
__device__ __forceinline__ unsigned long long draw_target(float u, unsigned long long s) {
  const double t = floor(double(u) * double(s));
  const unsigned long long v = t > 0.0 ? (unsigned long long)t : 0ull;
  return v < s ? v : s - 1;
}

template <typename T, bool kResident>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  constexpr int VEC = Logit<T>::kVec;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  uint32_t* list_key = reinterpret_cast<uint32_t*>(dyn);  // CTA 0: the remaining entries in index order
  uint32_t* list_idx = list_key + kList;
  // CTA 0's sort buffer; it lies over the row, which is no longer read then
  unsigned long long* sorted = reinterpret_cast<unsigned long long*>(dyn + kList * 8);
  float* xs = reinterpret_cast<float*>(dyn + kList * 8);  // this CTA's part of the row

  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int row = int(blockIdx.x) / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // the part of the row this CTA holds, in 16-byte granules of memory: slot s is entry first + s
  const char* base = a.logits + int64_t(row) * a.row_stride;
  const int lead = int((reinterpret_cast<uintptr_t>(base) & 15u) / sizeof(T));
  const int total_g = int((int64_t(lead) + a.vocab + VEC - 1) / VEC);
  const int g0 = int(int64_t(total_g) * rank / C), g1 = int(int64_t(total_g) * (rank + 1) / C);
  const int n_slots = (g1 - g0) * VEC;
  const int first = g0 * VEC - lead;
  auto granule = [&](int g, float* f) {  // entries of granule g of this part; those outside the row: -inf
    const int i0 = first + g * VEC;
    if (i0 >= 0 && i0 + VEC <= a.vocab) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(base + int64_t(i0) * int64_t(sizeof(T))));
      Logit<T>::unpack(u, f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = no_nan(f[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int i = i0 + j;
        f[j] = i >= 0 && i < a.vocab ? no_nan(Logit<T>::one(base + int64_t(i) * int64_t(sizeof(T)))) : kNegInf;
      }
    }
  };

  float tmax = kNegInf;
#pragma unroll 4
  for (int g = tid; g < g1 - g0; g += kThreads) {
    float f[VEC];
    granule(g, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) tmax = fmaxf(tmax, f[j]);
    if constexpr (kResident) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4)
        *reinterpret_cast<float4*>(xs + g * VEC + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
    }
  }
  const float temperature = a.temperature ? __ldg(a.temperature + row) : a.temperature_s;
  int k = a.top_k ? __ldg(a.top_k + row) : a.top_k_s;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p_s;
  const float min_p = fminf(a.min_p ? __ldg(a.min_p + row) : a.min_p_s, 1.f);
  const float u = __ldg(a.uniform + row);
  const bool greedy = !(temperature > 0.f);
  if (greedy) k = 1;
  const bool use_k = k > 0 && k < a.vocab;
  const bool use_p = top_p < 1.f;

  // the CTA's maximum, and its ceil(k / C)-th largest per-thread maximum
  const int k_part = (k + C - 1) / C;
  const bool use_tau = use_k && k_part <= kThreads / 4;
  {
    uint32_t lo = ordered(tmax), hi = lo;
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      sh.warp_count[warp] = lo;
      sh.warp_mass[warp] = hi;
    }
    __syncthreads();
    lo = sh.warp_count[lane & (kWarps - 1)];
    hi = uint32_t(sh.warp_mass[lane & (kWarps - 1)]);
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (tid == 0) sh.cta_max = from_ordered(hi);
    if (use_tau && k_part == 1) {
      lo = hi;
    } else if (use_tau) {
      // k_part threads reach lo throughout, so stopping early only loosens the bound
      const uint32_t mine = ordered(tmax);
      for (int it = 0; it < 20 && lo < hi; ++it) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        if (__syncthreads_count(mine >= mid) >= k_part) lo = mid;
        else hi = mid - 1;
      }
    }
    if (tid == 0) sh.cta_tau = from_ordered(lo);
  }
  cluster.sync();
  Scale sc;
  float tau = INFINITY;
  sc.m = kNegInf;
  for (int c = 0; c < C; ++c) {
    const Shared* o = cluster.map_shared_rank(&sh, c);
    sc.m = fmaxf(sc.m, o->cta_max);
    tau = fminf(tau, o->cta_tau);
  }
  if (k == 1) tau = sc.m;
  sc.greedy = greedy;
  sc.inv = greedy ? 0.f : 1.f / temperature;
  if (sc.m == kNegInf) {  // nothing can be drawn
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = kNegInf;
    }
    cluster.sync();  // no CTA leaves while another may read its memory
    return;
  }

  // warp w owns slots [w0, w1), four consecutive ones a lane and step, so warps hold rising indices
  const int per = ((n_slots + kWarps - 1) / kWarps + 127) & ~127;
  const int w0 = min(warp * per, n_slots), w1 = min(w0 + per, n_slots);
  auto load4 = [&](int s, float* f) {  // slots s .. s + 3 (s a multiple of 4); past the part: -inf
    if constexpr (kResident) {
      if (s < w1) {
        const float4 v = *reinterpret_cast<const float4*>(xs + s);
        f[0] = v.x;
        f[1] = v.y;
        f[2] = v.z;
        f[3] = v.w;
        return;
      }
      f[0] = f[1] = f[2] = f[3] = kNegInf;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = first + s + j;
        f[j] = s < w1 && i >= 0 && i < a.vocab ? no_nan(Logit<T>::one(base + int64_t(i) * int64_t(sizeof(T)))) : kNegInf;
      }
    }
  };

  // ---- which entries remain: x >= tau, or coarse bins up to `last_bin`; n of them in all
  bool listed = false;
  int last_bin = -1;
  unsigned long long total = 0;  // the row's whole mass, where it is known
  if (use_tau) {
    listed = true;
  } else if (use_k || use_p) {
    for (int i = tid; i < kBins; i += kThreads) {
      sh.hist_count[i] = 0;
      sh.hist_mass[i] = 0;
    }
    __syncthreads();
    unsigned long long sum = 0;
    for (int s = w0 + lane * 4; s < w1; s += 128) {
      float f[4];
      load4(s, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float z = sc.z(f[j]);
        const uint32_t w = weight(expf(z));
        sum += w;
        const float b = fabsf(z) * kBinScale;
        if (b < float(kBins)) {
          atomicAdd(&sh.hist_count[int(b)], 1u);
          atomicAdd(&sh.hist_mass[int(b)], (unsigned long long)w);
        }
      }
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.warp_mass[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      unsigned long long m = 0;
      for (int w = 0; w < kWarps; ++w) m += sh.warp_mass[w];
      sh.mass = m;
    }
    cluster.sync();
    if (warp == 0) {
      unsigned long long all = 0, m0 = 0, m1 = 0;
      uint32_t c0 = 0, c1 = 0;
      for (int c = 0; c < C; ++c) {
        const Shared* o = cluster.map_shared_rank(&sh, c);
        all += o->mass;
        c0 += o->hist_count[2 * lane];
        c1 += o->hist_count[2 * lane + 1];
        m0 += o->hist_mass[2 * lane];
        m1 += o->hist_mass[2 * lane + 1];
      }
      const uint32_t cs = warp_scan(c0 + c1, lane);
      const unsigned long long ms = warp_scan(m0 + m1, lane);
      // the first bin by which k entries, or the nucleus of the whole row, are reached
      bool at0, at1;
      if (use_k) {
        at0 = cs - c1 >= uint32_t(k);
        at1 = cs >= uint32_t(k);
      } else {
        const unsigned long long need = mass_needed(top_p, all);
        at0 = ms - m1 >= need;
        at1 = ms >= need;
      }
      const uint32_t has = __ballot_sync(0xffffffffu, at1);
      if (lane == 0) {
        sh.r0 = 0xffffffffu;
        sh.r1 = 0xffffffffu;
        sh.r2 = all;
      }
      __syncwarp();
      if (has != 0 && lane == __ffs(has) - 1) {
        sh.r0 = uint32_t(2 * lane + (at0 ? 0 : 1));
        sh.r1 = at0 ? cs - c1 : cs;
      }
    }
    __syncthreads();
    total = sh.r2;
    if (sh.r1 <= uint32_t(kList)) {
      listed = true;
      last_bin = int(sh.r0);
    }
    cluster.sync();  // everyone has read the bins
  }

  auto remains = [&](float x) -> bool {
    return last_bin < 0 ? (x >= tau && x > kNegInf) : fabsf(sc.z(x)) * kBinScale < float(last_bin + 1);
  };
  uint32_t n_all = 0;
  if (listed) {
    uint32_t mine = 0;
    for (int s = w0 + lane * 4; s < w1; s += 128) {
      float f[4];
      load4(s, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += remains(f[j]) ? 1u : 0u;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sh.warp_count[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      uint32_t n = 0;
      for (int w = 0; w < kWarps; ++w) n += sh.warp_count[w];
      sh.count = n;
    }
    cluster.sync();
    uint32_t before = 0;
    for (int c = 0; c < C; ++c) {
      const uint32_t n = cluster.map_shared_rank(&sh, c)->count;
      before += c < rank ? n : 0;
      n_all += n;
    }
    listed = n_all <= uint32_t(kList);
    if (listed && mine != 0) {  // to CTA 0's list, in index order
      for (int w = 0; w < warp; ++w) before += sh.warp_count[w];
      uint32_t* keys = cluster.map_shared_rank(list_key, 0);
      uint32_t* idxs = cluster.map_shared_rank(list_idx, 0);
      for (int s0 = w0; s0 < w1; s0 += 128) {
        float f[4];
        load4(s0 + lane * 4, f);
        uint32_t here = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) here |= remains(f[j]) ? 1u << j : 0u;
        if (__ballot_sync(0xffffffffu, here != 0) == 0) continue;
        const uint32_t incl = warp_scan(uint32_t(__popc(here)), lane);
        uint32_t at = before + incl - __popc(here);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (here >> j & 1u) {
            keys[at] = key_of(sc.z(f[j]));
            idxs[at] = uint32_t(first + s0 + lane * 4 + j);
            ++at;
          }
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    cluster.sync();
  }

  if (listed) {
    if (rank != 0) return;  // CTA 0 reads only its own memory from here on
    const int n = int(n_all);
    int np = 32;
    while (np < n) np <<= 1;
    for (int i = tid; i < np; i += kThreads)
      sorted[i] = i < n ? (uint64_t(list_key[i]) << 32) | uint32_t(i) : ~0ull;
    __syncthreads();
    for (int size = 2; size <= np; size <<= 1) {
      for (int stride = size >> 1; stride > 0; stride >>= 1) {
        for (int p = tid; p < np / 2; p += kThreads) {
          const int i = (p / stride) * stride * 2 + (p & (stride - 1)), j = i + stride;
          const bool up = (i & size) == 0;
          const unsigned long long x = sorted[i], y = sorted[j];
          if ((x > y) == up) {
            sorted[i] = y;
            sorted[j] = x;
          }
        }
        __syncthreads();
      }
    }
    // falling z: the weights' running sums, four neighbours a thread
    constexpr int kPer = kList / kThreads;
    unsigned long long w[kPer], sum = 0;
    float e[kPer];
    const int n_k = use_k ? min(k, n) : n;  // entries top-k leaves
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = tid * kPer + j;
      e[j] = i < n_k ? expf(z_of(uint32_t(sorted[i] >> 32))) : 0.f;
      w[j] = weight(e[j]);
      sum += w[j];
    }
    unsigned long long run = warp_scan(sum, lane);
    if (lane == 31) sh.warp_mass[warp] = run;
    __syncthreads();
    unsigned long long whole = 0;
    for (int x = 0; x < kWarps; ++x) {
      const unsigned long long m = sh.warp_mass[x];
      run += x < warp ? m : 0;
      whole += m;
    }
    run -= sum;
    // without top-k the list may be the row's upper part only, so its whole mass is `total`
    const unsigned long long need = use_p ? mass_needed(top_p, use_k ? whole : total) : ~0ull;
    uint32_t kept = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      kept += tid * kPer + j < n_k && run < need && !(e[j] < min_p) ? 1u : 0u;
      run += w[j];
    }
    kept = __reduce_add_sync(0xffffffffu, kept);
    if (lane == 0) sh.warp_count[warp] = kept;
    __syncthreads();
    kept = 0;
    for (int x = 0; x < kWarps; ++x) kept += sh.warp_count[x];
    const unsigned long long cut = sorted[kept - 1];  // the entry with z = 0 always stays
    __syncthreads();
    // rising index: the kept weights' running sum, and the first to pass the target
    sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = tid * kPer + j;
      const bool in = i < n && ((uint64_t(list_key[i]) << 32) | uint32_t(i)) <= cut;
      w[j] = in ? weight(expf(z_of(list_key[i]))) : 0;
      sum += w[j];
    }
    run = warp_scan(sum, lane);
    if (lane == 31) sh.warp_mass[warp] = run;
    __syncthreads();
    whole = 0;
    for (int x = 0; x < kWarps; ++x) {
      const unsigned long long m = sh.warp_mass[x];
      run += x < warp ? m : 0;
      whole += m;
    }
    run -= sum;
    const unsigned long long target = draw_target(u, whole);
    if (run <= target && target < run + sum) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (run <= target && target < run + w[j]) {
          const int i = tid * kPer + j;
          a.tokens[row] = int64_t(list_idx[i]);
          if (a.logprobs) a.logprobs[row] = z_of(list_key[i]) - logf(float(double(whole) / double(kUnit)));
        }
        run += w[j];
      }
    }
    return;
  }

  // ---- the cut by a radix search: entries with key < cut_key stay, and of those equal to it the first
  // `cut_ties` by index
  uint32_t cut_key = kDead, cut_ties = 0xffffffffu;
  if (use_k || use_p) {
    unsigned long long goal = use_k ? (unsigned long long)k : mass_needed(top_p, total);
    bool by_count = use_k;
    for (int search = 0; search < 2; ++search) {
      if (search == 1 && !(use_k && use_p)) break;
      uint32_t prefix = 0;
      unsigned long long below_n = 0, below_m = 0;  // entries and mass with smaller keys than `prefix`
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < kDigits; i += kThreads) {
          sh.hist_count[i] = 0;
          sh.hist_mass[i] = 0;
        }
        __syncthreads();
        const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int s = w0 + lane * 4; s < w1; s += 128) {
          float f[4];
          load4(s, f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = first + s + j;
            const float z = sc.z(f[j]);
            const uint32_t key = key_of(z);
            if (i >= 0 && i < a.vocab && (key & high) == prefix) {
              const uint32_t d = (key >> shift) & 255u;
              atomicAdd(&sh.hist_count[d], 1u);
              const uint32_t w = weight(expf(z));
              if (w != 0) atomicAdd(&sh.hist_mass[d], (unsigned long long)w);
            }
          }
        }
        cluster.sync();
        if (warp < kDigits / 32) {  // bins over the cluster, running sums over the digits
          unsigned long long m = 0;
          uint32_t n = 0;
          for (int c = 0; c < C; ++c) {
            const Shared* o = cluster.map_shared_rank(&sh, c);
            n += o->hist_count[tid];
            m += o->hist_mass[tid];
          }
          const uint32_t ns = warp_scan(n, lane);
          const unsigned long long ms = warp_scan(m, lane);
          cluster.sync();  // everyone has read the bins
          sh.hist_count[tid] = ns;
          sh.hist_mass[tid] = ms;
        } else {
          cluster.sync();
        }
        __syncthreads();
        if (tid == 0) {  // the first digit whose running sum reaches the goal
          unsigned long long n = below_n, m = below_m;
          int d = 0;
          bool found = false;
          for (int w = 0; w < kDigits / 32 && !found; ++w) {
            const unsigned long long wn = sh.hist_count[w * 32 + 31], wm = sh.hist_mass[w * 32 + 31];
            if ((by_count ? n + wn : m + wm) >= goal) {
              unsigned long long pn = 0, pm = 0;
              for (d = w * 32; d < w * 32 + 31; ++d) {
                const unsigned long long dn = sh.hist_count[d], dm = sh.hist_mass[d];
                if ((by_count ? n + dn : m + dm) >= goal) break;
                pn = dn;
                pm = dm;
              }
              n += pn;
              m += pm;
              found = true;
            } else {
              n += wn;
              m += wm;
            }
          }
          if (!found) d = kDigits - 1;
          sh.r0 = uint32_t(d);
          sh.r2 = n;
          sh.r3 = m;
        }
        __syncthreads();
        prefix |= sh.r0 << shift;
        below_n = sh.r2;
        below_m = sh.r3;
        __syncthreads();
      }
      const unsigned long long w = weight(expf(z_of(prefix)));
      unsigned long long ties;
      if (by_count) ties = goal - below_n;
      else ties = w != 0 ? (goal - below_m + w - 1) / w : 0xffffffffull;
      if (ties > 0xffffffffull) ties = 0xffffffffull;
      // a nucleus lies within the top k: where both end at one key, the smaller part stays
      if (search == 1 && prefix == cut_key && ties > cut_ties) ties = cut_ties;
      cut_key = prefix;
      cut_ties = uint32_t(ties);
      if (search == 0 && use_k && use_p) {
        goal = mass_needed(top_p, below_m + w * ties);
        by_count = false;
      }
    }
    cluster.sync();
  }

  // ---- walk the row: where this CTA's and this warp's ties begin, then the kept mass
  const bool limit_ties = cut_ties != 0xffffffffu;
  uint32_t tie0 = 0;
  if (limit_ties) {
    uint32_t mine = 0;
    for (int s = w0 + lane * 4; s < w1; s += 128) {
      float f[4];
      load4(s, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = first + s + j;
        mine += i >= 0 && i < a.vocab && key_of(sc.z(f[j])) == cut_key ? 1u : 0u;
      }
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sh.warp_count[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      uint32_t n = 0;
      for (int w = 0; w < kWarps; ++w) n += sh.warp_count[w];
      sh.ties = n;
    }
    cluster.sync();
    for (int c = 0; c < rank; ++c) tie0 += cluster.map_shared_rank(&sh, c)->ties;
    for (int w = 0; w < warp; ++w) tie0 += sh.warp_count[w];
  }
  // the kept weights of this lane's four slots; advances the warp's tie count
  auto kept4 = [&](int s, uint32_t& ties, uint32_t* w) {
    float f[4];
    load4(s, f);
    uint32_t key[4], tie = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = first + s + j;
      const float z = sc.z(f[j]), e = expf(z);
      key[j] = key_of(z);
      const bool in = i >= 0 && i < a.vocab && key[j] <= cut_key && !(e < min_p);
      w[j] = in ? weight(e) : 0u;
      tie |= i >= 0 && i < a.vocab && key[j] == cut_key ? 1u << j : 0u;
    }
    if (limit_ties && __ballot_sync(0xffffffffu, tie != 0) != 0) {
      const uint32_t incl = warp_scan(uint32_t(__popc(tie)), lane);
      uint32_t at = ties + incl - __popc(tie);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (tie >> j & 1u) {
          if (at >= cut_ties) w[j] = 0;
          ++at;
        }
      }
      ties += __shfl_sync(0xffffffffu, incl, 31);
    }
  };
  {
    unsigned long long sum = 0;
    uint32_t ties = tie0;
    for (int s0 = w0; s0 < w1; s0 += 128) {
      uint32_t w[4];
      kept4(s0 + lane * 4, ties, w);
      sum += (unsigned long long)w[0] + w[1] + w[2] + w[3];
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.warp_mass[warp] = sum;
  }
  __syncthreads();
  if (tid == 0) {
    unsigned long long m = 0;
    for (int w = 0; w < kWarps; ++w) m += sh.warp_mass[w];
    sh.mass = m;
  }
  cluster.sync();
  unsigned long long whole = 0, before = 0;
  for (int c = 0; c < C; ++c) {
    const unsigned long long m = cluster.map_shared_rank(&sh, c)->mass;
    before += c < rank ? m : 0;
    whole += m;
  }
  const unsigned long long target = draw_target(u, whole);
  for (int w = 0; w < warp; ++w) before += sh.warp_mass[w];
  if (before <= target && target < before + sh.warp_mass[warp]) {
    uint32_t ties = tie0;
    for (int s0 = w0; s0 < w1; s0 += 128) {
      uint32_t w[4];
      kept4(s0 + lane * 4, ties, w);
      const unsigned long long sum = (unsigned long long)w[0] + w[1] + w[2] + w[3];
      const unsigned long long incl = warp_scan(sum, lane);
      unsigned long long run = before + incl - sum;
      if (run <= target && target < run + sum) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (run <= target && target < run + w[j]) {
            const int i = first + s0 + lane * 4 + j;
            a.tokens[row] = i;
            if (a.logprobs) {
              const float z = sc.z(no_nan(Logit<T>::one(base + int64_t(i) * int64_t(sizeof(T)))));
              a.logprobs[row] = z - logf(float(double(whole) / double(kUnit)));
            }
          }
          run += w[j];
        }
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      if (before > target) break;
    }
  }
  cluster.sync();  // no CTA leaves while another may read its memory
}

template <typename T, bool kResident>
int launch(const SampleArgs& a, int rows, int cluster, size_t smem, cudaStream_t st) {
  using augur_kv_dev::fail;
  static size_t attr_bytes[augur_kv_dev::kMaxDevices] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= augur_kv_dev::kMaxDevices)
    return fail(AUGUR_KV_ECUDA, "sample: cannot query the current device");
  {
    std::lock_guard<std::recursive_mutex> lock(augur_kv_dev::g_cache_mutex);
    if (attr_bytes[dev] < smem) {
      if (cudaFuncSetAttribute(sample_kernel<T, kResident>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) !=
          cudaSuccess)
        return augur_kv_dev::check_launch("cudaFuncSetAttribute(sample_kernel)");
      attr_bytes[dev] = smem;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows) * unsigned(cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(cluster);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, kResident>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(AUGUR_KV_ECUDA, "sample_kernel: %s", cudaGetErrorString(e));
  }
  return AUGUR_KV_OK;
}

}  // namespace augur_kv_smp

#define AUGUR_KV_EXPORT extern "C" __attribute__((visibility("default")))

AUGUR_KV_EXPORT int augur_kv_sample(const void* logits, int64_t row_stride, int32_t rows, int32_t vocab,
                                    int32_t dtype, const float* uniform, const float* temperature,
                                    float temperature_all, const int32_t* top_k, int32_t top_k_all,
                                    const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                                    int64_t* tokens, float* logprobs, void* stream) {
  using namespace augur_kv_smp;
  using augur_kv_dev::fail;
  augur_kv_dev::g_last_error[0] = '\0';
  const int es = augur_kv_dev::elem_size(dtype);
  if (es == 0) return fail(AUGUR_KV_EINVAL, "sample: unknown dtype %d", dtype);
  if (rows < 0 || vocab <= 0 || vocab > (1 << 21)) return fail(AUGUR_KV_EINVAL, "sample: bad sizes");
  if (rows == 0) return AUGUR_KV_OK;
  if (logits == nullptr || uniform == nullptr || tokens == nullptr)
    return fail(AUGUR_KV_EINVAL, "sample: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(logits) & uintptr_t(es - 1)) != 0 || rows > 1 << 24)
    return fail(AUGUR_KV_EINVAL, "sample: logits must be aligned to their type, and rows at most 2^24");
  SampleArgs a;
  memset(&a, 0, sizeof(a));
  a.logits = static_cast<const char*>(logits);
  a.row_stride = row_stride * es;
  a.vocab = vocab;
  a.uniform = uniform;
  a.temperature = temperature;
  a.temperature_s = temperature_all;
  a.top_k = top_k;
  a.top_k_s = top_k_all;
  a.top_p = top_p;
  a.top_p_s = top_p_all;
  a.min_p = min_p;
  a.min_p_s = min_p_all;
  a.tokens = tokens;
  a.logprobs = logprobs;
  // CTAs per row: as many as keep the GPU's resident CTAs (two an SM) busy, at
  // least enough for the row to fit their shared memory, and parts of at
  // least 2,048 entries
  const int vec = 16 / es;
  constexpr size_t kMost = 200 * 1024;  // of the 227 KB a CTA may have
  auto bytes = [&](int c) {
    const int64_t granules = ((int64_t(vocab) + vec - 1) / vec + 1 + c - 1) / c;
    const size_t part = size_t(granules) * size_t(vec) * 4;
    return size_t(kList) * 8 + (part > size_t(kList) * 8 ? part : size_t(kList) * 8);
  };
  const int64_t slots = int64_t(augur_kv_dev::sm_count()) * 2;
  int c = 1;
  while (c < kMaxCluster && (bytes(c) > kMost / 2 || (int64_t(rows) * c * 2 <= slots * 2 && vocab / (c * 2) >= 2048))) c *= 2;
  const bool resident = bytes(c) <= kMost;
  const size_t smem = resident ? bytes(c) : size_t(kList) * 16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AUGUR_KV_F32)
    return resident ? launch<float, true>(a, rows, c, smem, st) : launch<float, false>(a, rows, c, smem, st);
  if (dtype == AUGUR_KV_F16)
    return resident ? launch<__half, true>(a, rows, c, smem, st) : launch<__half, false>(a, rows, c, smem, st);
  return resident ? launch<__nv_bfloat16, true>(a, rows, c, smem, st)
                  : launch<__nv_bfloat16, false>(a, rows, c, smem, st);
}
