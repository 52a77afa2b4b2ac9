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
// rate); the rest is the latency of a handful of cluster exchanges and, where
// many entries are in question, of shared-memory additions.
//  * A row belongs to a cluster of 1 to 8 CTAs; each copies its part of the row
//    to shared memory (cp.async), so HBM is read once and every later pass
//    runs from there. Parts too long for that are read again, from L2 mostly.
//  * Top-k: the per-thread maxima, binned by |z|, bound the k-th largest (at
//    least k entries reach the bin by which k maxima are counted). The few
//    entries at or above that bin go to a list, in any order, which CTA 0 of the
//    cluster sorts twice: by z, to cut it, and what stays by index, to draw.
//  * Top-p: the mass within a few depths of the maximum tells between which two
//    the nucleus ends; a histogram between these (512 bins of masses) shows the
//    bin. Where the nucleus is likely to fit the list, it goes there; else the
//    entries of that bin alone do (after further histograms where they are too
//    many), CTA 0 finds the key at which the nucleus ends and how many of its
//    ties belong to it, and the draw walks the row in place. Top-k takes this
//    way too, with counts, where its own bound leaves too many.
//  * With neither, the draw walks the row at once; greedy rows look for the
//    lowest index of the maximum only.
//  * Values are cut in the logits' own order: a key's limit becomes the smallest
//    x below it (found by looking around the rounded inverse), so the passes
//    compare x and take no exponential of what is not kept.
// Measured (B200, warm): 1 row of 151,936 bf16: top-k 50 16 us, top-p 0.95 45 us
// (60 us before the searches looked near a guess, one addition served a warp
// and the cut was found by bins, not by sorting), greedy 10 us; 256 rows of
// float32 (156 MB, floor 24 us): greedy 62 us, top-k 50 84 us, top-p 0.95 349 us.

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
constexpr int kList = 2048;  // most entries CTA 0 sorts
constexpr int kBins = kThreads;  // bins of a histogram, one a thread
constexpr float kBinScale = kBins / 21.6f;  // linear bins of |z|: e^-21.6 has no weight any more
constexpr int kDepths = 5;  // of the maximum at which top-p first looks
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
};

// What the CTAs of a cluster tell one another (each writes its own copy).
struct Shared {
  float cta_max;
  uint32_t first;  // greedy: the lowest index of the maximum
  uint32_t count, ties;
  unsigned long long mass;
  uint32_t warp_count[kWarps];
  unsigned long long warp_mass[kWarps];
  // histogram; masses in halves of 16 bits (a part has at most 65,536 entries), or whole where it has more
  uint32_t bin_count[kBins], bin_lo[kBins], bin_hi[kBins];
  unsigned long long bin_mass[kBins];
  unsigned long long depth_mass[kWarps][kDepths + 1], cta_depth_mass[kDepths + 1];  // within depths of the maximum, and in all
  // results of a step, written by one thread; cut: by CTA 0 for the cluster
  uint32_t found, found_n;
  unsigned long long found_m;
  uint32_t cut_key, cut_same;
  unsigned long long cut_n, cut_mass;
};

template <typename T> struct Logit;
template <> struct Logit<float> {
  static constexpr int kVec = 4;  // entries of 16 bytes
  static constexpr uint32_t kLowest = 0xff800000u;  // -inf, as stored
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
  static constexpr uint32_t kLowest = 0xff80ff80u;
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
  static constexpr uint32_t kLowest = 0xfc00fc00u;
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
  float m, inv;
  __device__ __forceinline__ float z(float x) const {
    const float v = fmaxf((x - m) * inv, kNegInf);  // a NaN (of the row's, or -inf * 0): dead
    return x == m ? 0.f : v;                        // inf - inf
  }
};
__device__ __forceinline__ uint32_t key_of(float z) { return __float_as_uint(fabsf(z)); }
__device__ __forceinline__ float z_of(uint32_t key) { return -__uint_as_float(key); }
__device__ __forceinline__ uint32_t weight(float e) { return __float2uint_rz(e * kUnit); }

// Of masses, below 2^54 each: halves of 27 bits, which 32 of cannot pass 32 bits.
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
  const uint32_t low = __reduce_add_sync(0xffffffffu, uint32_t(v) & 0x7ffffffu);
  return low + ((unsigned long long)__reduce_add_sync(0xffffffffu, uint32_t(v >> 27)) << 27);
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

// Bins of equal width over |z|, from a depth on. Rising in |z|; below 0 before that depth.
struct Bins {
  float start, scale;
  __device__ __forceinline__ float of(float z) const { return (fabsf(z) - start) * scale; }
};
// The smallest value in [lo, hi) for which `pred`, which turns true once, holds (hi if none). A warp
// tries 32 values a step.
template <typename F>
__device__ __forceinline__ uint32_t first_true(uint32_t lo, uint32_t hi, F pred) {
  const uint32_t lane = threadIdx.x & 31;
  while (lo < hi) {
    const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;  // lane 0 tries lo, the last ones may pass hi
    const uint32_t yes = __ballot_sync(0xffffffffu, at >= hi || at < lo || pred(at));
    const uint32_t f = yes ? uint32_t(__ffs(yes)) - 1 : 32u;
    if (f == 0) return lo;
    const uint32_t below = lo + (f - 1) * step;  // false there
    if (f < 32 && below < hi - step) hi = lo + f * step;  // true there
    lo = below + 1;
  }
  return hi;
}
// The same, looking around a guess first: two steps where it is within 512, seven where it is not.
template <typename F>
__device__ __forceinline__ uint32_t first_true_near(uint32_t guess, uint32_t lo, uint32_t hi, F pred) {
  const uint32_t base = guess > lo + 512u ? guess - 512u : lo, at = base + (threadIdx.x & 31) * 32;
  const uint32_t yes = __ballot_sync(0xffffffffu, at >= hi || at < base || pred(at));
  if (yes != 0 && ((yes & 1u) == 0 || base == lo)) {
    const uint32_t f = uint32_t(__ffs(yes)) - 1;
    return f == 0 ? lo : first_true(base + (f - 1) * 32 + 1, min(base + f * 32, hi), pred);
  }
  return first_true(lo, hi, pred);
}
// The smallest key whose bin is b or above.
__device__ __noinline__ uint32_t bin_edge(Bins bins, int b) {
  return first_true_near(__float_as_uint(bins.start + float(b) / bins.scale), 0u, kDead,
                         [&](uint32_t key) { return bins.of(__uint_as_float(key)) >= float(b); });
}

// CTA-wide running sums, inclusive.
__device__ __noinline__ uint32_t scan_count(Shared& sh, uint32_t n) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t cum = warp_scan(n, lane);
  if (lane == 31) sh.warp_count[warp] = cum;
  __syncthreads();
  cum += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_count[lane] : 0u);
  __syncthreads();
  return cum;
}
__device__ __noinline__ unsigned long long scan_mass(Shared& sh, unsigned long long m) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long cum = warp_scan(m, lane);
  if (lane == 31) sh.warp_mass[warp] = cum;
  __syncthreads();
  cum += warp_sum(lane < warp ? sh.warp_mass[lane] : 0ull);
  __syncthreads();
  return cum;
}

// Sorts n entries (at most kList) in place, rising. Their bin is the high word (a float's bits, or a whole
// number) times `scale`; they find their bin's place, then their rank in the bin by comparing.
__device__ __noinline__ void sort_entries(Shared& sh, unsigned long long* list, int n, bool floats, float scale) {
  constexpr int kPer = kList / kThreads;
  const int tid = threadIdx.x;
  unsigned long long e[kPer];
  int b[kPer];
  sh.bin_count[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid + j * kThreads;
    b[j] = -1;
    if (i < n) {
      e[j] = list[i];
      const uint32_t high = uint32_t(e[j] >> 32);
      b[j] = min(int((floats ? __uint_as_float(high) : float(high)) * scale), kBins - 1);
      atomicAdd(&sh.bin_count[b[j]], 1u);
    }
  }
  __syncthreads();
  const uint32_t c = sh.bin_count[tid];
  const uint32_t cum = scan_count(sh, c);
  sh.bin_lo[tid] = cum - c;  // the bin's first place
  sh.bin_hi[tid] = 0;        // of it taken
  __syncthreads();
  uint32_t place[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (b[j] >= 0) {
      place[j] = sh.bin_lo[b[j]] + atomicAdd(&sh.bin_hi[b[j]], 1u);
      list[place[j]] = e[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (b[j] < 0) continue;
    const uint32_t start = sh.bin_lo[b[j]], count = sh.bin_count[b[j]];
    uint32_t rank = 0;  // entries are unlike
    for (uint32_t x = start; x < start + count; ++x) rank += list[x] < e[j] ? 1u : 0u;
    place[j] = start + rank;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (b[j] >= 0) list[place[j]] = e[j];
  __syncthreads();
}

// The smallest x with a key below `end`, up to the maximum (keys fall as x rises; the maximum's is 0).
__device__ __noinline__ float x_below(Scale sc, uint32_t end) {
  const float guess = sc.m - __uint_as_float(end) / sc.inv;
  return from_ordered(first_true_near(ordered(guess == guess ? guess : sc.m), ordered(kNegInf), ordered(sc.m),
                                      [&](uint32_t o) { return key_of(sc.z(from_ordered(o))) < end; }));
}

template <typename T, bool kResident>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a) {
  constexpr int VEC = Logit<T>::kVec;
  constexpr int kStep = 32 * VEC;  // slots a warp takes at a time
  constexpr int kPer = kList / kThreads;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  // entries in question, (key, index); CTA 0's hold the cluster's
  unsigned long long* list = reinterpret_cast<unsigned long long*>(dyn);
  unsigned char* part = dyn + kList * 8;  // this CTA's part of the row, as stored

  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int row = int(blockIdx.x) / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // every CTA's value of one field, a lane each (lanes past the cluster: `none`): one exchange's latency, not C of them
  auto of_lane = [&](auto field, auto none) { return lane < C ? field(*cluster.map_shared_rank(&sh, lane)) : none; };
  // the sum over the cluster of one field for each thread: the loads go out together
  auto cluster_sum = [&](auto field) {
    decltype(field(sh)) v[kMaxCluster];
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) v[c] = c < C ? field(*cluster.map_shared_rank(&sh, c)) : 0;
    auto sum = v[0];
#pragma unroll
    for (int c = 1; c < kMaxCluster; ++c) sum += v[c];
    return sum;
  };

  // the part of the row this CTA holds, in 16-byte granules of memory: slot s is entry first + s
  const char* base = a.logits + int64_t(row) * a.row_stride;
  const int lead = int((reinterpret_cast<uintptr_t>(base) & 15u) / sizeof(T));
  const int total_g = int((int64_t(lead) + a.vocab + VEC - 1) / VEC);
  const int g0 = int(int64_t(total_g) * rank / C), g1 = int(int64_t(total_g) * (rank + 1) / C);
  const int n_g = g1 - g0, n_slots = n_g * VEC;
  const int first = g0 * VEC - lead;
  const char* part_base = base + int64_t(first) * int64_t(sizeof(T));  // 16-byte aligned
  // granules that lie in the row whole: [in0, in1)
  const int in0 = first < 0 ? 1 : 0, in1 = first + n_slots > a.vocab ? n_g - 1 : n_g;
  auto edge_granule = [&](int g) -> uint4 {  // entries outside the row: -inf
    uint4 u = make_uint4(Logit<T>::kLowest, Logit<T>::kLowest, Logit<T>::kLowest, Logit<T>::kLowest);
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int i = first + g * VEC + j;
      if (i >= 0 && i < a.vocab) e[j] = reinterpret_cast<const T*>(base)[i];
    }
    return u;
  };
  if constexpr (kResident) {
    for (int g = tid; g < n_g; g += kThreads) {
      if (g >= in0 && g < in1) {
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(part + g * 16));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(part_base + int64_t(g) * 16) : "memory");
      } else {
        *reinterpret_cast<uint4*>(part + g * 16) = edge_granule(g);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  auto granule = [&](int g, float* f) {
    uint4 u;
    if constexpr (kResident) u = *reinterpret_cast<const uint4*>(part + g * 16);
    else u = g >= in0 && g < in1 ? __ldg(reinterpret_cast<const uint4*>(part_base + int64_t(g) * 16)) : edge_granule(g);
    Logit<T>::unpack(u, f);
  };
  // All granules of the part, a thread every kThreads-th (the ones it copied itself), several loads under way. The
  // lanes of a warp take each step together; those past the part see entries of -inf.
  auto each_granule = [&](auto use) {
    constexpr int kBatch = kResident ? 2 : 8;
    const uint4 none = make_uint4(Logit<T>::kLowest, Logit<T>::kLowest, Logit<T>::kLowest, Logit<T>::kLowest);
    float f[VEC];
    for (int s0 = warp * 32; s0 < n_g; s0 += kBatch * kThreads) {
      uint4 u[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int g = s0 + i * kThreads + lane;
        if constexpr (kResident) u[i] = g < n_g ? *reinterpret_cast<const uint4*>(part + g * 16) : none;
        else u[i] = g >= in0 && g < in1 ? __ldg(reinterpret_cast<const uint4*>(part_base + int64_t(g) * 16)) : none;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i > 0 && s0 + i * kThreads >= n_g) break;
        Logit<T>::unpack(u[i], f);
        use(s0 + i * kThreads + lane, f);
      }
    }
    if (!kResident && warp == 0) {  // those that lie in the row in part: the first and the last
      const int g = lane == 0 && in0 > 0 ? 0 : lane == 1 && in1 < n_g && n_g > in0 ? n_g - 1 : -1;
      Logit<T>::unpack(g >= 0 ? edge_granule(g) : none, f);
      use(g, f);
    }
  };
  const float temperature = a.temperature ? __ldg(a.temperature + row) : a.temperature_s;
  int k = a.top_k ? __ldg(a.top_k + row) : a.top_k_s;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p_s;
  const float min_p_given = a.min_p ? __ldg(a.min_p + row) : a.min_p_s;
  const float min_p = min_p_given > 0.f ? fminf(min_p_given, 1.f) : 0.f;
  const float u = __ldg(a.uniform + row);

  float tmax = kNegInf;  // fmaxf passes NaN over
  each_granule([&](int, const float* f) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) tmax = fmaxf(tmax, f[j]);
  });
  {
    float m = tmax;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sh.warp_count[warp] = __float_as_uint(m);
    sh.bin_count[tid] = 0;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) m = fmaxf(m, __uint_as_float(sh.warp_count[w]));
      sh.cta_max = m;
    }
  }
  cluster.sync();
  Scale sc;
  sc.m = of_lane([](const Shared& o) { return o.cta_max; }, kNegInf);
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) sc.m = fmaxf(sc.m, __shfl_xor_sync(0xffffffffu, sc.m, o));
  sc.m = __shfl_sync(0xffffffffu, sc.m, 0);
  const bool greedy = !(temperature > 0.f);
  sc.inv = greedy ? 0.f : 1.f / temperature;
  if (greedy) k = 1;
  bool use_k = k > 0 && k < a.vocab;
  const bool use_p = top_p < 1.f;
  if (sc.m == kNegInf) {  // nothing can be drawn
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = kNegInf;
    }
    cluster.sync();  // no CTA leaves while another may read its memory
    return;
  }

  // warp w owns slots [w0, w1), VEC consecutive ones a lane and step, so warps hold rising indices
  const int per = ((n_slots + kWarps - 1) / kWarps + kStep - 1) / kStep * kStep;
  const int w0 = min(warp * per, n_slots), w1 = min(w0 + per, n_slots);
  // Slots s .. s + VEC - 1 (whole granules); past the warp's: -inf. A NaN stays one: it lies in no bin and no key
  // range, and its weight is 0 (a conversion to a whole number takes NaN to 0).
  auto load = [&](int s, float* f) {
    if (s < w1) {
      granule(s / VEC, f);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = kNegInf;
    }
  };

  if (k == 1) {  // the lowest index of the maximum
    uint32_t best = 0xffffffffu;
    for (int g = tid; g < n_g && best == 0xffffffffu; g += kThreads) {
      float f[VEC];
      granule(g, f);
#pragma unroll
      for (int j = VEC - 1; j >= 0; --j)
        if (f[j] == sc.m) best = uint32_t(first + g * VEC + j);
    }
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0) sh.warp_count[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) best = min(best, sh.warp_count[w]);
      sh.first = best;
    }
    cluster.sync();
    if (rank == 0 && warp == 0) {
      best = __reduce_min_sync(0xffffffffu, of_lane([](const Shared& o) { return o.first; }, 0xffffffffu));
      if (lane == 0) {
        a.tokens[row] = int64_t(best);
        if (a.logprobs) a.logprobs[row] = 0.f;
      }
    }
    cluster.sync();
    return;
  }

  const Bins all_bins = {0.f, kBinScale};
  // ---- the bins up to `last_bin` hold all that can be drawn, if they fit the list
  int last_bin = -1;
  unsigned long long total = 0;  // the row's mass, where it is known
  if (use_k) {  // per-thread maxima: k of them reach this bin, so k entries do
    const float b = all_bins.of(sc.z(tmax));
    if (b < float(kBins)) atomicAdd(&sh.bin_count[int(b)], 1u);
    cluster.sync();
    const uint32_t n = cluster_sum([&](const Shared& o) { return o.bin_count[tid]; });
    if (tid == 0) sh.found = kBins;
    const uint32_t cum_n = scan_count(sh, n);
    if (cum_n >= uint32_t(k) && cum_n - n < uint32_t(k)) sh.found = uint32_t(tid);
    __syncthreads();
    if (sh.found < uint32_t(kBins)) last_bin = int(sh.found);
    else cluster.sync();  // everyone has read the bins
  }

  // Entries with x in [low, high) (all up to the maximum where `open`), into CTA 0's list in any order.
  // Returns how many there are in the cluster, or some number above kList; only where they fit (kList) is the
  // list filled, and only in CTA 0.
  auto collect = [&](float low, float high, bool open) -> uint32_t {
    if (tid == 0) sh.count = 0;
    __syncthreads();
    each_granule([&](int g, const float* f) {
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) bits |= f[j] >= low && (open || f[j] < high) ? 1u << j : 0u;  // never a NaN
      const uint32_t lanes = __ballot_sync(0xffffffffu, bits != 0);
      if (lanes == 0) return;
      // additions to one word wait for one another: from many lanes, one for all
      const uint32_t mine = uint32_t(__popc(bits));
      uint32_t at = 0;
      if (__popc(lanes) <= 6) {
        if (bits != 0) at = atomicAdd(&sh.count, mine);
      } else {
        const uint32_t incl = warp_scan(mine, lane);
        if (lane == 31) at = atomicAdd(&sh.count, incl);
        at = __shfl_sync(0xffffffffu, at, 31) + incl - mine;
      }
      if (bits == 0 || at >= uint32_t(kList)) return;  // too many: how many does not matter
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (bits >> j & 1u) {
          if (at < uint32_t(kList)) list[at] = (uint64_t(key_of(sc.z(f[j]))) << 32) | uint32_t(first + g * VEC + j);
          ++at;
        }
      }
    });
    cluster.sync();
    const uint32_t theirs = of_lane([](const Shared& o) { return o.count; }, 0u);
    const uint32_t ends = warp_scan(theirs, lane);  // of the CTAs' entries, in the list
    const uint32_t n_all = __shfl_sync(0xffffffffu, ends, kMaxCluster - 1);
    if (n_all <= uint32_t(kList) && rank == 0) {
      for (uint32_t i0 = __shfl_sync(0xffffffffu, theirs, 0); i0 < n_all; i0 += kThreads) {
        const uint32_t i = i0 + tid;
        int c = 0;
        uint32_t start = 0;
#pragma unroll
        for (int x = 0; x < kMaxCluster - 1; ++x) {
          const uint32_t end = __shfl_sync(0xffffffffu, ends, x);
          if (i >= end && x < C - 1) {
            c = x + 1;
            start = end;
          }
        }
        if (i < n_all) list[i] = cluster.map_shared_rank(list, c)[i - start];
      }
    }
    cluster.sync();
    return n_all;
  };
  // CTA 0: draws from the list, which holds all that can be drawn (keys below `end`), and writes the row's result.
  auto draw_from_list = [&](int n, uint32_t end) {
    sort_entries(sh, list, n, true, kBins / __uint_as_float(end));
    // falling z: the weights' running sums, kPer neighbours a thread
    unsigned long long w[kPer], sum = 0;
    float e[kPer];
    const int n_k = use_k ? min(k, n) : n;  // entries top-k leaves
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = tid * kPer + j;
      e[j] = i < n_k ? expf(z_of(uint32_t(list[i] >> 32))) : 0.f;
      w[j] = weight(e[j]);
      sum += w[j];
    }
    unsigned long long run = scan_mass(sh, sum);
    if (tid == kThreads - 1) sh.found_m = run;
    __syncthreads();
    // without top-k the list may be the row's upper part only: its whole mass is `total`
    const unsigned long long need = use_p ? mass_needed(top_p, use_k ? sh.found_m : total) : ~0ull;
    run -= sum;
    uint32_t kept = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      kept += tid * kPer + j < n_k && run < need && !(e[j] < min_p) ? 1u : 0u;
      run += w[j];
    }
    kept = scan_count(sh, kept);
    if (tid == kThreads - 1) sh.found = kept;
    __syncthreads();
    const int n_kept = int(sh.found);  // the first of the list: at least the entry with z = 0
    // by rising index: the kept weights' running sum, and the first to pass the target
    for (int i = tid; i < n_kept; i += kThreads) list[i] = (list[i] << 32) | (list[i] >> 32);
    __syncthreads();
    sort_entries(sh, list, n_kept, false, float(kBins) / float(a.vocab));
    sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = tid * kPer + j;
      w[j] = i < n_kept ? weight(expf(z_of(uint32_t(list[i])))) : 0;
      sum += w[j];
    }
    run = scan_mass(sh, sum);
    if (tid == kThreads - 1) sh.found_m = run;
    __syncthreads();
    const unsigned long long whole = sh.found_m, target = draw_target(u, whole);
    run -= sum;
    if (run <= target && target < run + sum) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (run <= target && target < run + w[j]) {
          const unsigned long long it = list[tid * kPer + j];
          a.tokens[row] = int64_t(it >> 32);
          if (a.logprobs) a.logprobs[row] = z_of(uint32_t(it)) - logf(float(double(whole) / double(kUnit)));
        }
        run += w[j];
      }
    }
  };
  auto list_up_to = [&](Bins bins, int bin) -> bool {  // true: the row is done
    const uint32_t end = bin_edge(bins, bin + 1);
    const uint32_t n = collect(x_below(sc, end), 0.f, true);
    if (n > uint32_t(kList)) return false;
    if (rank == 0) draw_from_list(int(n), end);  // from CTA 0's memory alone
    return true;
  };
  if (last_bin >= 0 && list_up_to(all_bins, last_bin)) return;

  // entries below the key stay, and of those at it (cut_same, or more than is known) the first cut_ties
  uint32_t cut_key = kDead, cut_ties = 0xffffffffu, cut_same = 0xffffffffu;
  if (use_k || use_p) {
    // Counts are kept where something is looked for by count, masses where something is by mass.
    auto add_to_bin = [&](bool counts, int b, uint32_t w) {
      if (counts) atomicAdd(&sh.bin_count[b], 1u);
      if (!use_p) return;
      if constexpr (kResident) {
        atomicAdd(&sh.bin_lo[b], w & 0xffffu);
        if (w >> 16) atomicAdd(&sh.bin_hi[b], w >> 16);
      } else {  // parts may be longer: carry by hand
        const uint32_t old = atomicAdd(&sh.bin_lo[b], w);
        if (old + w < old) atomicAdd(&sh.bin_hi[b], 1u);
      }
    };
    auto bin_mass = [&] { return (unsigned long long)sh.bin_lo[tid] + ((unsigned long long)sh.bin_hi[tid] << (kResident ? 16 : 32)); };
    // One histogram over the cluster: this thread's bin, and the running sums up to and with it.
    auto histogram = [&](bool counts, auto bin, uint32_t& n, unsigned long long& m, uint32_t& cum_n, unsigned long long& cum_m) {
      sh.bin_count[tid] = sh.bin_lo[tid] = sh.bin_hi[tid] = 0;
      __syncthreads();
      each_granule([&](int, const float* f) {
        int b[VEC];
        uint32_t w[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {  // without branches: the chains of the entries run beside one another
          const float z = sc.z(f[j]);
          b[j] = bin(f[j], z);
          w[j] = use_p ? weight(expf(z)) : 0u;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (b[j] >= 0) add_to_bin(counts, b[j], w[j]);
      });
      __syncthreads();
      sh.bin_mass[tid] = bin_mass();
      cluster.sync();
      n = cum_n = 0;
      m = cum_m = 0;
      if (counts) {
        n = cluster_sum([&](const Shared& o) { return o.bin_count[tid]; });
        cum_n = scan_count(sh, n);
      }
      if (use_p) {
        m = cluster_sum([&](const Shared& o) { return o.bin_mass[tid]; });
        cum_m = scan_mass(sh, m);
      }
      cluster.sync();  // everyone has read the bins
    };
    // The bin whose running sum is the first to reach the goal; what lies before it, and in it.
    auto find = [&](bool by_count, unsigned long long goal, uint32_t n, unsigned long long m, uint32_t cum_n,
                    unsigned long long cum_m, unsigned long long& below_n, unsigned long long& below_m) -> int {
      const unsigned long long c0 = by_count ? below_n + cum_n - n : below_m + cum_m - m;
      const unsigned long long c1 = by_count ? below_n + cum_n : below_m + cum_m;
      __syncthreads();
      if (c0 < goal && goal <= c1) {
        sh.found = uint32_t(tid);
        sh.found_n = uint32_t(below_n + cum_n - n);
        sh.found_m = below_m + cum_m - m;
      }
      __syncthreads();
      below_n = sh.found_n;
      below_m = sh.found_m;
      return int(sh.found);
    };
    // The exact cut within keys [lo, hi), behind below_n entries of mass below_m; leaves cut_key and
    // cut_ties and returns the mass up to the cut.
    auto refine = [&](bool by_count, unsigned long long goal, uint32_t lo, uint32_t hi, unsigned long long below_n,
                      unsigned long long below_m) __attribute__((always_inline)) -> unsigned long long {
      auto shift_of = [&] {
        int shift = 0;
        while ((hi - lo - 1) >> shift >= uint32_t(kBins)) ++shift;
        return shift;
      };
      auto narrow = [&](int shift, uint32_t n, unsigned long long m, uint32_t cum_n, unsigned long long cum_m) {
        const int b = find(by_count, goal, n, m, cum_n, cum_m, below_n, below_m);
        lo += uint32_t(b) << shift;
        hi = min(hi, lo + (1u << shift));
      };
      cut_same = 0xffffffffu;
      // by the cluster, until the list holds what is left or it is one key
      while (hi - lo > 1) {
        const uint32_t in_n = collect(x_below(sc, hi), lo == 0 ? 0.f : x_below(sc, lo), lo == 0);
        if (in_n <= uint32_t(kList)) {  // then by CTA 0 alone
          if (rank == 0) {
            while (hi - lo > 1) {
              const int shift = shift_of();
              sh.bin_count[tid] = sh.bin_lo[tid] = sh.bin_hi[tid] = 0;
              __syncthreads();
              for (uint32_t i = tid; i < in_n; i += kThreads) {
                const uint32_t key = uint32_t(list[i] >> 32);
                if (key >= lo && key < hi) add_to_bin(by_count, int((key - lo) >> shift), weight(expf(z_of(key))));
              }
              __syncthreads();
              const uint32_t n = sh.bin_count[tid];
              const unsigned long long m = bin_mass();
              narrow(shift, n, m, by_count ? scan_count(sh, n) : 0, use_p ? scan_mass(sh, m) : 0);
            }
            uint32_t same = 0;
            for (uint32_t i = tid; i < in_n; i += kThreads) same += uint32_t(list[i] >> 32) == lo ? 1u : 0u;
            same = scan_count(sh, same);
            if (tid == kThreads - 1) {
              sh.cut_key = lo;
              sh.cut_same = same;
              sh.cut_n = below_n;
              sh.cut_mass = below_m;
            }
          }
          cluster.sync();
          const Shared* o = cluster.map_shared_rank(&sh, 0);
          lo = o->cut_key;
          cut_same = o->cut_same;
          below_n = o->cut_n;
          below_m = o->cut_mass;
          cluster.sync();  // everyone has read the cut
          break;
        }
        const int shift = shift_of();
        uint32_t n, cum_n;
        unsigned long long m, cum_m;
        histogram(by_count, [&](float, float z) {
          const uint32_t key = key_of(z);
          return key >= lo && key < hi ? int((key - lo) >> shift) : -1;
        }, n, m, cum_n, cum_m);
        narrow(shift, n, m, cum_n, cum_m);
      }
      const unsigned long long w = weight(expf(z_of(lo)));
      const unsigned long long ties = by_count ? goal - below_n : w != 0 ? (goal - below_m + w - 1) / w : 1;
      cut_key = lo;
      cut_ties = uint32_t(ties);
      return below_m + w * ties;
    };

    uint32_t n, cum_n;
    unsigned long long m, cum_m;
    float from = kNegInf, to = INFINITY;  // the histogram takes entries in [from, to)
    unsigned long long above_m = 0;       // mass of those from `to` on, and the first key past theirs
    uint32_t above_key = 0;
    Bins bins = all_bins;
    if (!use_k) {
      // top-p alone: the row's mass, and between which depths the nucleus ends, so that the histogram's atomics
      // are spent on few entries
      const float depth[kDepths] = {3.f, 6.f, 9.f, 12.f, 15.f};
      unsigned long long sum[kDepths + 1] = {0, 0, 0, 0, 0, 0};
      each_granule([&](int, const float* f) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float z = sc.z(f[j]);
          const uint32_t w = weight(expf(z));
          sum[kDepths] += w;
#pragma unroll
          for (int d = 0; d < kDepths; ++d) sum[d] += z >= -depth[d] ? w : 0u;
        }
      });
#pragma unroll
      for (int d = 0; d <= kDepths; ++d) sum[d] = warp_sum(sum[d]);
      __syncthreads();
      if (lane == 0) {
#pragma unroll
        for (int d = 0; d <= kDepths; ++d) sh.depth_mass[warp][d] = sum[d];
      }
      __syncthreads();
      if (tid <= kDepths) {
        unsigned long long all = 0;
        for (int w = 0; w < kWarps; ++w) all += sh.depth_mass[w][tid];
        sh.cta_depth_mass[tid] = all;
      }
      cluster.sync();
#pragma unroll
      for (int d = 0; d <= kDepths; ++d) sum[d] = warp_sum(of_lane([&](const Shared& o) { return o.cta_depth_mass[d]; }, 0ull));
      total = sum[kDepths];
      const unsigned long long need = mass_needed(top_p, total);
      float end = 0.f, start = 0.f;  // depths
#pragma unroll
      for (int d = kDepths - 1; d >= 0; --d) {
        if (sum[d] >= need) end = depth[d];
        else if (start == 0.f) {
          start = depth[d];
          above_m = sum[d];
        }
      }
      // |z| in (start, end]: falling x
      if (end > 0.f) from = x_below(sc, __float_as_uint(end) + 1);
      if (start > 0.f) {
        above_key = __float_as_uint(start) + 1;
        to = x_below(sc, above_key);
      }
      // all the bins for this range (past 21.6, nothing has a weight): fewer entries meet in one
      bins.start = start;
      bins.scale = (float(kBins) - 0.5f) / ((end > 0.f ? end : 21.6f) - start);
    }
    histogram(use_k, [&](float x, float z) {
      const float b = bins.of(z);
      return x >= from && (x < to || to == INFINITY) && b < float(kBins) ? int(b) : -1;
    }, n, m, cum_n, cum_m);
    if (tid == kThreads - 1) {
      sh.found_n = cum_n;
      sh.found_m = cum_m;
    }
    __syncthreads();
    if (use_k) total = sh.found_m;
    use_k = use_k && sh.found_n > uint32_t(k);  // entries past the bins have no weight
    if (use_k || use_p) {
      unsigned long long below_n = 0, below_m = above_m;
      const unsigned long long goal = use_k ? (unsigned long long)k : mass_needed(top_p, total);
      const int b = find(use_k, goal, n, m, cum_n, cum_m, below_n, below_m);
      // with counts it is known whether the list will hold them; without, a nucleus that ends this side of e^-6 is tried
      if ((use_k ? below_n < (unsigned long long)kList : bins.of(9.f) > float(b)) && list_up_to(bins, b)) return;
      // a bin that holds the depth `start` begins, for the search, behind it
      const unsigned long long mass = refine(use_k, goal, max(bin_edge(bins, b), above_key), bin_edge(bins, b + 1), below_n, below_m);
      if (use_k && use_p) {
        const uint32_t k_key = cut_key, k_ties = cut_ties;
        const unsigned long long need = mass_needed(top_p, mass);
        below_n = below_m = 0;
        const int b2 = find(false, need, n, m, cum_n, cum_m, below_n, below_m);
        refine(false, need, bin_edge(bins, b2), bin_edge(bins, b2 + 1), below_n, below_m);
        // the nucleus lies within the top k: where both end at one key, the smaller part stays
        if (cut_key == k_key) cut_ties = min(cut_ties, k_ties);
      }
    }
  }

  // ---- walk the row: where this CTA's and this warp's ties begin, then the kept mass
  const bool limit_ties = cut_ties < cut_same;
  // entries below this are not kept, and only ties of those above: most of a warp's steps hold none of these
  const uint32_t none = first_true_near(__float_as_uint(fminf(21.5f, min_p > 0.f ? -logf(min_p) : 21.5f)), 0u, kDead, [&](uint32_t key) {
    const float e = expf(z_of(key));
    return e < min_p || weight(e) == 0;
  });
  const float x_cut = x_below(sc, cut_key < none ? cut_key + 1 : none);
  auto any_from = [&](const float* f) {
    float most = f[0];
#pragma unroll
    for (int j = 1; j < VEC; ++j) most = fmaxf(most, f[j]);
    return __any_sync(0xffffffffu, most >= x_cut);
  };
  uint32_t tie0 = 0;
  if (limit_ties) {
    uint32_t mine = 0;
    for (int s0 = w0; s0 < w1; s0 += kStep) {
      float f[VEC];
      load(s0 + lane * VEC, f);
      if (!any_from(f)) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) mine += key_of(sc.z(f[j])) == cut_key ? 1u : 0u;
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
    const uint32_t theirs = of_lane([](const Shared& o) { return o.ties; }, 0u);
    tie0 = __reduce_add_sync(0xffffffffu, lane < rank ? theirs : 0u) +
           __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_count[lane] : 0u);
  }
  // the kept weights of this lane's slots (an entry without weight is never kept); advances the warp's tie count
  auto kept = [&](int s, uint32_t& ties, uint32_t* w) -> unsigned long long {
    float f[VEC];
    load(s, f);
    unsigned long long sum = 0;
    if (!any_from(f)) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = 0;
      return 0;
    }
    if (!limit_ties) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const uint32_t x = weight(expf(sc.z(f[j])));
        w[j] = f[j] >= x_cut ? x : 0u;
        sum += w[j];
      }
      return sum;
    }
    uint32_t tie = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float z = sc.z(f[j]);
      const uint32_t x = weight(expf(z));
      w[j] = f[j] >= x_cut ? x : 0u;
      tie |= key_of(z) == cut_key ? 1u << j : 0u;
    }
    if (__ballot_sync(0xffffffffu, tie != 0) != 0) {
      const uint32_t incl = warp_scan(uint32_t(__popc(tie)), lane);
      uint32_t at = ties + incl - __popc(tie);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (tie >> j & 1u) {
          if (at >= cut_ties) w[j] = 0;
          ++at;
        }
      }
      ties += __shfl_sync(0xffffffffu, incl, 31);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += w[j];
    return sum;
  };
  {
    unsigned long long sum = 0;
    uint32_t ties = tie0;
    for (int s0 = w0; s0 < w1; s0 += kStep) {
      uint32_t w[VEC];
      sum += kept(s0 + lane * VEC, ties, w);
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
  const unsigned long long theirs = of_lane([](const Shared& o) { return o.mass; }, 0ull);
  const unsigned long long whole = warp_sum(theirs), target = draw_target(u, whole);
  unsigned long long before = warp_sum((lane < rank ? theirs : 0ull) + (lane < warp ? sh.warp_mass[lane] : 0ull));
  if (before <= target && target < before + sh.warp_mass[warp]) {
    uint32_t ties = tie0;
    for (int s0 = w0; s0 < w1; s0 += kStep) {
      uint32_t w[VEC];
      const unsigned long long sum = kept(s0 + lane * VEC, ties, w);
      const unsigned long long incl = warp_scan(sum, lane);
      unsigned long long run = before + incl - sum;
      if (run <= target && target < run + sum) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (run <= target && target < run + w[j]) {
            const int i = first + s0 + lane * VEC + j;
            a.tokens[row] = i;
            if (a.logprobs) {
              const float z = sc.z(Logit<T>::one(base + int64_t(i) * int64_t(sizeof(T))));
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
  // CTAs per row: as many as the GPU holds at once (two an SM), at least 4 (a row whose nucleus is wide takes
  // long, and with fewer CTAs a batch waits for it: 256 rows of 151,936 float32 logits with mixed settings take 205 us
  // with 2, 167 with 4, 183 with 8), with parts of at least 2,048 entries. Parts stay in shared memory where two
  // CTAs' fit an SM's; else every pass reads them again, from L2 for the most part.
  const int vec = 16 / es;
  constexpr size_t kMost = 100 * 1024;  // of the 227 KB an SM's CTAs may have
  auto bytes = [&](int c) {  // the list and the part
    const int64_t granules = ((int64_t(vocab) + vec - 1) / vec + 1 + c - 1) / c;
    return size_t(kList) * 8 + size_t(granules) * 16;
  };
  const int64_t slots = int64_t(augur_kv_dev::sm_count()) * 2;
  int c = 1;
  while (c < kMaxCluster && vocab / (c * 2) >= 2048 && (c < 4 || int64_t(rows) * c * 2 <= slots)) c *= 2;
  // masses are added in halves of 16 bits: a part has at most 65,536 entries
  const bool resident = bytes(c) <= kMost && (vocab + 2 * vec) / c + vec <= 65536;
  const size_t smem = resident ? bytes(c) : size_t(kList) * 8;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AUGUR_KV_F32)
    return resident ? launch<float, true>(a, rows, c, smem, st) : launch<float, false>(a, rows, c, smem, st);
  if (dtype == AUGUR_KV_F16)
    return resident ? launch<__half, true>(a, rows, c, smem, st) : launch<__half, false>(a, rows, c, smem, st);
  return resident ? launch<__nv_bfloat16, true>(a, rows, c, smem, st)
                  : launch<__nv_bfloat16, false>(a, rows, c, smem, st);
}
