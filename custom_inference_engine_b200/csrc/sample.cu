// A sampled token per row of fp16 logits: temperature, top-k, top-p, min-p and the
// inverse of the cumulative distribution at a given random number.
//
// The tokens kept by each of the three filters are a prefix of the row sorted by
// logit, and the sampled token is the one at which the cumulative mass of that
// order crosses u * (kept mass). fp16 has 2^16 values, so the sorted row is its
// histogram over the 2^16 ordered keys: the counts are whole numbers (exact
// whatever the order of the atomics), a key's weight exp((value - max) / T) is
// taken once per key that occurs, and masses are fp64 sums in a fixed order. So the
// token depends on nothing but the inputs. The row is read twice and never sorted.
//
// One cluster of C CTAs per row, C parts of the row:
//   1. every CTA counts its part into 2^16 16-bit counters in its shared memory
//      (two to a word, 128 KiB; a part has at most 65528 tokens, so none overflows);
//   2. the keys form 256 chunks of 256; warps sum a chunk's counters over the
//      cluster (distributed shared memory) and hand CTA 0 the chunk's tokens,
//      mass and tokens that min-p keeps;
//   3. CTA 0's first warp finds the kept prefix and the key of the sampled token
//      with its rank among the tokens of that key, descending into one chunk for
//      each prefix;
//   4. the CTA whose part holds that token looks it up in the row.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cie_host.h"
#include "cie_model_ops.h"

namespace cie {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kKeys = 1 << 16;
constexpr int kChunks = 256;              // of 256 keys, 8 per lane
constexpr int kMaxPart = 65528;           // tokens of a part: multiple of 8 below 2^16
constexpr int kMaxCluster = 8;
constexpr unsigned int kMinusInf = 0xFC00;  // key of -inf; key 0 is NaN, 0x3FF +inf

struct Params {
  const __half* logits;
  int64_t stride;
  const float* uniform;
  const float* temperature;
  const int64_t* top_k;     // may be null, as top_p and min_p
  const float* top_p;
  const float* min_p;
  int64_t* out;
  int vocab;
  int part;                 // tokens per CTA, multiple of 8
  int vec;                  // rows start on 16-byte boundaries
};

struct Shared {
  uint32_t hist[kKeys / 2];       // counter of key d: half d & 1 of word d >> 1
  double mass[kChunks];           // CTA 0: per chunk
  int count[kChunks];
  int above[kChunks];             // tokens with w >= min_p
  int warp_sum[kThreads / 32];
  unsigned int top;               // smallest key (largest logit) of this CTA's part
  unsigned int key;               // the sampled token's key and its rank among the
  int rank;                       // row's tokens of that key
};

// Ordered key of a fp16 value: 0 for NaN, then descending values; -0 and +0 share one.
__device__ __forceinline__ unsigned int key_of(unsigned int bits) {
  if ((bits & 0x7fffu) > 0x7c00u) return 0u;
  if (bits == 0x8000u) bits = 0u;
  return (bits & 0x8000u) ? bits : 0x7fffu - bits;
}

__device__ __forceinline__ double value_of(unsigned int key) {
  const unsigned int bits = key >= 0x8000u ? key : 0x7fffu - key;
  return static_cast<double>(__half2float(__ushort_as_half(static_cast<unsigned short>(bits))));
}

__device__ __forceinline__ double weight(unsigned int key, unsigned int top, double peak,
                                         double temp) {
  if (key == top) return 1.0;
  if (key >= kMinusInf) return 0.0;
  return exp((value_of(key) - peak) / temp);
}

// Counters of keys [8 j, 8 j + 8) summed over the cluster.
__device__ __forceinline__ void counts8(cg::cluster_group& cluster, Shared* sh, int parts, int j,
                                        int (&c)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = 0;
  for (int r = 0; r < parts; ++r) {
    const uint4 u = reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh->hist, r))[j];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[2 * e] += static_cast<int>(w[e] & 0xffffu);
      c[2 * e + 1] += static_cast<int>(w[e] >> 16);
    }
  }
}

// f(index, key) over the tokens [lo, hi), 8 to a load where rows are aligned.
template <typename F>
__device__ __forceinline__ void each_key(const Params& p, const __half* row, int lo, int hi, F&& f) {
  const int n8 = p.vec ? (hi - lo) >> 3 : 0;  // lo is a multiple of 8
  for (int i = threadIdx.x; i < n8; i += kThreads) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + lo + 8 * i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f(lo + 8 * i + 2 * e, key_of(w[e] & 0xffffu));
      f(lo + 8 * i + 2 * e + 1, key_of(w[e] >> 16));
    }
  }
  for (int i = lo + 8 * n8 + threadIdx.x; i < hi; i += kThreads)
    f(i, key_of(__half_as_ushort(row[i])));
}

__device__ __forceinline__ double warp_scan(double v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// n as a number of tokens, 1 .. c (a NaN gives 1).
__device__ __forceinline__ int whole(double n, int c) {
  return n >= c ? c : n > 1.0 ? static_cast<int>(n) : 1;
}

// A place in the row's sorted order: `tokens` tokens of total mass `mass` come
// before rank `rank` of key `key`.
struct Place {
  int tokens;
  double mass;
  unsigned int key;
  int rank;
};

// The search of one row, by one warp of CTA 0.
struct Search {
  cg::cluster_group& cluster;
  Shared* sh;
  int parts, lane;
  unsigned int top;
  double peak, temp;

  // The last token whose preceding tokens satisfy `before(tokens, mass)`, a
  // predicate that holds for nothing before and fails from some place on. Chunks,
  // then lanes of a chunk, then keys, then tokens of a key (their number from
  // `within(tokens, mass, weight, count)`, 1 .. count).
  template <typename Before, typename Within>
  __device__ Place last(Before before, Within within) const {
    // chunk: lane holds 8 neighbouring ones
    int tok[8], sum_t = 0;
    double mass[8], sum_m = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      tok[e] = sh->count[8 * lane + e];
      mass[e] = sh->mass[8 * lane + e];
      sum_t += tok[e];
      sum_m += mass[e];
    }
    int t = warp_scan(sum_t, lane) - sum_t;
    double m = warp_scan(sum_m, lane) - sum_m;
    if (lane == 0) m = 0.0;
    int best = -1, best_t = 0;
    double best_m = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (tok[e] > 0 && (t == 0 || before(t, m))) {
        best = 8 * lane + e;
        best_t = t;
        best_m = m;
      }
      t += tok[e];
      m += mass[e];
    }
    const int chunk = __reduce_max_sync(0xffffffffu, best);
    const int from = chunk >> 3;
    best_t = __shfl_sync(0xffffffffu, best_t, from);
    best_m = __shfl_sync(0xffffffffu, best_m, from);
    // keys of the chunk: lane holds 8
    int c[8];
    double w[8];
    counts8(cluster, sh, parts, chunk * 32 + lane, c);
    sum_t = 0;
    sum_m = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = c[e] > 0 ? weight(chunk * 256 + 8 * lane + e, top, peak, temp) : 0.0;
      sum_t += c[e];
      sum_m += c[e] * w[e];
    }
    t = best_t + warp_scan(sum_t, lane) - sum_t;
    m = best_m + (warp_scan(sum_m, lane) - sum_m);
    if (lane == 0) m = best_m;
    best = -1;
    int best_c = 0;
    double best_w = 0.0;
    int bt = 0;
    double bm = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (c[e] > 0 && (t == best_t || before(t, m))) {
        best = 8 * lane + e;
        best_c = c[e];
        best_w = w[e];
        bt = t;
        bm = m;
      }
      t += c[e];
      m += c[e] * w[e];
    }
    const int k = __reduce_max_sync(0xffffffffu, best);
    const int src = k >> 3;
    bt = __shfl_sync(0xffffffffu, bt, src);
    bm = __shfl_sync(0xffffffffu, bm, src);
    best_c = __shfl_sync(0xffffffffu, best_c, src);
    best_w = __shfl_sync(0xffffffffu, best_w, src);
    const int r = min(max(within(bt, bm, best_w, best_c), 1), best_c) - 1;
    return Place{bt + r, bm + r * best_w, static_cast<unsigned int>(chunk * 256 + k), r};
  }

  // The token of rank n - 1 (n >= 1), with the mass before it.
  __device__ Place nth(int n) const {
    return last([=](int t, double) { return t < n; },
                [=](int t, double, double, int) { return n - t; });
  }
};

__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared* sh = reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks());
  const int part = static_cast<int>(cluster.block_rank());
  const int64_t r = blockIdx.x / parts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const __half* row = p.logits + r * p.stride;
  const int lo = static_cast<int>(min(static_cast<int64_t>(part) * p.part, static_cast<int64_t>(p.vocab)));
  const int hi = min(lo + p.part, p.vocab);

  // ---- 1. histogram of this part ------------------------------------------------
  for (int i = threadIdx.x; i < kKeys / 8; i += kThreads)
    reinterpret_cast<uint4*>(sh->hist)[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) sh->top = kKeys;
  __syncthreads();
  unsigned int top = kKeys;
  each_key(p, row, lo, hi, [&](int, unsigned int key) {
    top = min(top, key);
    atomicAdd(&sh->hist[key >> 1], (key & 1u) ? 0x10000u : 1u);
  });
  top = __reduce_min_sync(0xffffffffu, top);
  if (lane == 0) atomicMin(&sh->top, top);
  cluster.sync();
  for (int q = 0; q < parts; ++q) top = min(top, *cluster.map_shared_rank(&sh->top, q));

  const float t32 = p.temperature[r];
  const bool greedy = !(t32 > 0.f) || top == 0u || top >= kMinusInf;  // uniform over the cluster
  const double peak = value_of(top), temp = static_cast<double>(t32);
  if (!greedy) {
    // ---- 2. tokens and mass of every chunk of keys -------------------------------
    const double min_p = p.min_p ? static_cast<double>(p.min_p[r]) : 0.0;
    Shared* sh0 = cluster.map_shared_rank(sh, 0);
    for (int ch = part * (kThreads / 32) + warp; ch < kChunks; ch += parts * (kThreads / 32)) {
      int c[8], n = 0, above = 0;
      double m = 0.0;
      counts8(cluster, sh, parts, ch * 32 + lane, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (c[e] > 0) {
          const double w = weight(ch * 256 + 8 * lane + e, top, peak, temp);
          n += c[e];
          m += c[e] * w;
          if (w >= min_p && w > 0.0) above += c[e];
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      n = __reduce_add_sync(0xffffffffu, n);
      above = __reduce_add_sync(0xffffffffu, above);
      if (lane == 0) {
        sh0->mass[ch] = m;
        sh0->count[ch] = n;
        sh0->above[ch] = above;
      }
    }
    cluster.sync();
  }

  // ---- 3. the sampled token's key and rank ---------------------------------------
  if (part == 0 && warp == 0) {
    unsigned int key = top;
    int rank = 0;
    if (!greedy) {
      const Search s{cluster, sh, parts, lane, top, peak, temp};
      int above = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) above += sh->above[8 * lane + e];
      int kept = max(__reduce_add_sync(0xffffffffu, above), 1);
      const int64_t k = p.top_k ? p.top_k[r] : 0;
      int n_k = k > 0 && k < p.vocab ? static_cast<int>(k) : p.vocab;
      const double top_p = p.top_p ? static_cast<double>(p.top_p[r]) : 1.0;
      if (top_p < 1.0) {
        // mass of the top-k prefix, then the ranks whose preceding mass is below
        // top_p of it
        const Place z = s.nth(n_k);
        const double all = z.mass + weight(z.key, top, peak, temp);
        const double target = top_p * all;
        const Place q = s.last([=](int, double m) { return m < target; },
                               [=](int, double m, double w, int c) {
                                 return whole(ceil((target - m) / w), c);
                               });
        n_k = min(n_k, q.tokens + 1);
      }
      kept = min(kept, n_k);
      const Place z = s.nth(kept);
      const double target = static_cast<double>(p.uniform[r]) *
                            (z.mass + weight(z.key, top, peak, temp));
      // the last token with no more than the target before it
      Place q = s.last([=](int, double m) { return m <= target; },
                       [=](int, double m, double w, int c) {
                         return whole(floor((target - m) / w) + 1.0, c);
                       });
      if (q.tokens >= kept) q = z;
      key = q.key;
      rank = q.rank;
    }
    if (lane < parts) {
      Shared* to = cluster.map_shared_rank(sh, lane);
      to->key = key;
      to->rank = rank;
    }
  }
  cluster.sync();

  // ---- 4. its index: the rank-th token with that key -------------------------------
  const unsigned int key = sh->key;
  int rank = sh->rank;
  auto counter = [&](int q) {
    const uint32_t w = *cluster.map_shared_rank(&sh->hist[key >> 1], q);
    return static_cast<int>((key & 1u) ? w >> 16 : w & 0xffffu);
  };
  for (int q = 0; q < part; ++q) rank -= counter(q);
  const int own = counter(part);
  cluster.sync();  // no CTA leaves while another reads its counters
  if (rank < 0 || rank >= own) return;
  // contiguous tokens per thread, in order
  const int each = (hi - lo + kThreads - 1) / kThreads;
  const int a = min(lo + static_cast<int>(threadIdx.x) * each, hi), z = min(a + each, hi);
  int n = 0;
  for (int i = a; i < z; ++i) n += key_of(__half_as_ushort(row[i])) == key;
  int before = warp_scan(n, lane) - n;
  if (lane == 31) sh->warp_sum[warp] = before + n;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += sh->warp_sum[w];
  if (rank >= before && rank < before + n) {
    for (int i = a; i < z; ++i) {
      if (key_of(__half_as_ushort(row[i])) == key && before++ == rank) {
        p.out[r] = i;
        break;
      }
    }
  }
}

}  // namespace sample
}  // namespace cie

extern "C" {

int cie_sample_rows(const void* logits, int64_t rows, int64_t vocab, int64_t stride,
                    const float* uniform, const float* temperature, const int64_t* top_k,
                    const float* top_p, const float* min_p, int64_t* out, cie_stream_t stream) {
  using namespace cie;
  using namespace cie::sample;
  if (rows < 0 || vocab < 0) return fail(CIE_ERR_INVALID_ARGUMENT, "negative size");
  if (rows == 0) return CIE_OK;
  if (!logits || !uniform || !temperature || !out || vocab == 0)
    return fail(CIE_ERR_INVALID_ARGUMENT, "null pointer or empty row");
  if (vocab > static_cast<int64_t>(kMaxPart) * kMaxCluster)
    return fail(CIE_ERR_UNSUPPORTED, "vocab %lld > %d", (long long)vocab, kMaxPart * kMaxCluster);
  if (stride < vocab) return fail(CIE_ERR_INVALID_ARGUMENT, "row stride < vocab");
  if ((reinterpret_cast<uintptr_t>(logits) & 1) != 0)
    return fail(CIE_ERR_ALIGNMENT, "logits must be 2-byte aligned");
  // parts a row needs, and more while every CTA still finds an SM of its own
  int parts = 1;
  auto part_of = [&](int c) { return (vocab + 8LL * c - 1) / (8LL * c) * 8; };
  while (part_of(parts) > kMaxPart) parts *= 2;
  while (parts < kMaxCluster && rows * parts * 2 <= sm_count() && part_of(parts) > 4096) parts *= 2;
  if (rows > 0x7fffffff / kMaxCluster) return fail(CIE_ERR_OVERFLOW, "too many rows");
  Params p;
  p.logits = static_cast<const __half*>(logits);
  p.stride = stride;
  p.uniform = uniform;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.out = out;
  p.vocab = static_cast<int>(vocab);
  p.part = static_cast<int>(part_of(parts));
  p.vec = aligned16(logits) && stride % 8 == 0;
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(&sample_kernel),
                                       static_cast<int>(sizeof(Shared)), 5);
  if (st != CIE_OK) return st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, p);
  if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
  return CIE_OK;
}

}  // extern "C"
