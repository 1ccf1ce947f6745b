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

constexpr int kThreads = 512;
constexpr int kKeys = 1 << 16;
constexpr int kChunks = 256;              // of 256 keys, 8 per lane
constexpr int kMaxPart = 65528;           // tokens of a part: multiple of 8 below 2^16
constexpr int kMaxCluster = 8;
// keys of some values
constexpr unsigned int kPlusInf = 0x3FF, kFirstFinite = 0x400, kPlusZero = 0x7FFF;
constexpr unsigned int kMinusZero = 0x8000, kMinusInf = 0xFC00;

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
};

struct alignas(16) Shared {
  uint32_t hist[kKeys / 2];       // counter of key d: half d & 1 of word d >> 1
  // CTA 0, per chunk: mass and tokens, those of all chunks before, and those that min-p
  // keeps (`some` says that it drops any)
  double mass[kChunks], mass_before[kChunks], mass_above[kChunks];
  int count[kChunks], before[kChunks], above[kChunks];
  int some;
  int warp_sum[kThreads / 32];
  unsigned int top, bottom;       // smallest and largest key of this CTA's part
  unsigned int tops[kMaxCluster], bottoms[kMaxCluster];  // and of every part
  unsigned int key;               // the sampled token's key and its rank among this
  int rank;                       // part's tokens of that key (negative: not here)
};

// Ordered keys of two fp16 values: descending values ascend, NaNs lie below +inf's key
// and above -inf's, -0 (0x8000) comes after +0 (0x7fff).
__device__ __forceinline__ uint32_t keys_of2(uint32_t bits) {
  return bits ^ ((~bits >> 15 & 0x00010001u) * 0x7fffu);  // 0x7fff - b for positive b
}

// The key under which a token is looked up: one for -0 and +0, one (0) for every NaN.
__device__ __forceinline__ unsigned int key_of(unsigned int bits) {
  if ((bits & 0x7fffu) > 0x7c00u) return 0u;
  if (bits == 0x8000u) bits = 0u;
  return (bits & 0x8000u) ? bits : 0x7fffu - bits;
}

// 2^e for -1022 <= e <= 1023.
__device__ __forceinline__ double exp2_of(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// The number of tokens c (below 2^32) as a double.
__device__ __forceinline__ double as_double(unsigned int c) {
  return __hiloint2double(0x43300000, static_cast<int>(c)) - 4503599627370496.0;
}

// fp16 value of a finite key, and the step (< 0) to the next key's value in its binade
// of 1024 keys.
__device__ __forceinline__ double value_of(unsigned int key, double& step) {
  const unsigned int bits = key >= 0x8000u ? key : 0x7fffu - key;
  const int binade = static_cast<int>(bits >> 10 & 31u);
  const unsigned int whole = (bits & 1023u) + (binade ? 1024u : 0u);
  const double ulp = exp2_of(max(binade, 1) - 25);
  step = -ulp;
  return as_double(whole) * ((bits & 0x8000u) ? -ulp : ulp);
}

// exp(x) for -700 <= x <= 0, without a branch, so that several run interleaved: x =
// k ln 2 + r with |r| <= ln 2 / 2 (ln 2 in two parts, after Cody and Waite), 2^k in the
// exponent and the Taylor series of exp(r) through r^13, whose remainder is below 2^-57.
__device__ __forceinline__ double exp_above_700(double x) {
  constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is k
  const double t = fma(x, 1.4426950408889634, kShift), k = t - kShift;
  const double r = fma(k, -2.3190468138462996e-17, fma(k, -0.6931471805599453, x));
  const double r2 = r * r, r4 = r2 * r2;
  const double a = fma(r2, fma(r, 1.0 / 6, 0.5), fma(r, 1.0, 1.0));
  const double b = fma(r2, fma(r, 1.0 / 5040, 1.0 / 720), fma(r, 1.0 / 120, 1.0 / 24));
  const double c = fma(r2, fma(r, 1.0 / 39916800, 1.0 / 3628800), fma(r, 1.0 / 362880, 1.0 / 40320));
  const double d = fma(r, 1.0 / 6227020800, 1.0 / 479001600);
  const double p = fma(r4, fma(r4, fma(r4, d, c), b), a);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

// The weights of neighbouring keys of one binade: key first + e weighs
// base * ratio^(e - shift) from e = shift on and nothing before, where shift > 0 only
// if first lies above the row's largest logit. Two exponentials for 8 or 32 weights,
// each within 2^-47 of exp((value - peak) / temp).
struct Weights {
  double base;
  int shift;
  bool tiny;  // some of the keys may weigh 0: take base from Scale::exact
};

struct Scale {
  unsigned int top;      // the row's smallest key
  double peak, inv_temp; // its value, 1 / temperature

  // the weights of two neighbouring keys of first's binade, one by the other
  __device__ __forceinline__ double ratio(unsigned int first) const {
    double step;
    value_of(first, step);
    const double x = step * inv_temp;
    return top < kFirstFinite || first >= kMinusInf || x < -700.0 ? 0.0 : exp_above_700(fmax(x, -700.0));
  }

  __device__ __forceinline__ Weights from(unsigned int first, double keys = 8.0) const {
    const unsigned int at = max(first, top);
    double step;
    const double x = (value_of(at, step) - peak) * inv_temp;
    // all of the weight is the largest logit's when that is +inf; -inf has none
    const bool tiny = !(fma(keys * step, inv_temp, x) > -700.0) || top < kFirstFinite ||
                      first >= kMinusInf;
    return Weights{exp_above_700(tiny ? -700.0 : x), static_cast<int>(at - first), tiny};
  }

  __device__ __forceinline__ double exact(unsigned int first) const {
    const unsigned int at = max(first, top);
    if (at == top) return 1.0;
    if (top < kFirstFinite || first >= kMinusInf) return 0.0;
    double step;
    return exp((value_of(at, step) - peak) * inv_temp);
  }
};

// Counters of keys [8 j, 8 j + 8) summed over the cluster, from part `first` on (each
// part begins with its own, so that no part is read by all at once).
template <int kParts>
__device__ __forceinline__ void counts8(cg::cluster_group& cluster, Shared* sh, int first, int j,
                                        unsigned int (&c)[8]) {
  uint4 u[kParts];
#pragma unroll
  for (int r = 0; r < kParts; ++r)
    u[r] = reinterpret_cast<const uint4*>(
        cluster.map_shared_rank(sh->hist, (first + r) % kParts))[j];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = 0;
#pragma unroll
  for (int r = 0; r < kParts; ++r) {
    const uint32_t w[4] = {u[r].x, u[r].y, u[r].z, u[r].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // low and high half added in one instruction each
      c[2 * e] = __dp2a_lo(w[e], 0x0001u, c[2 * e]);
      c[2 * e + 1] = __dp2a_lo(w[e], 0x0100u, c[2 * e + 1]);
    }
  }
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

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What is asked of the sorted order. Every query holds of the first token and fails from
// some place on: fewer than `count` tokens come before, or a mass below `mass` does
// (up to `mass`, with `or_equal`).
struct Query {
  bool by_count, or_equal;
  int count;
  double mass;

  __device__ __forceinline__ bool before(int t, double m) const {
    return by_count ? t < count : or_equal ? m <= mass : m < mass;
  }
  // how many of a key's c tokens, w each, behind t tokens of mass m (1 .. c; 1 for a NaN)
  __device__ __forceinline__ int within(int t, double m, double w, int c) const {
    const double q = (mass - m) / w;
    const double n = by_count ? static_cast<double>(count - t) : or_equal ? floor(q) + 1.0 : ceil(q);
    return n >= c ? c : n > 1.0 ? static_cast<int>(n) : 1;
  }
};

// A token of the row's sorted order: `tokens` tokens of total mass `mass` come
// before it; it is number `rank` of key `key`'s tokens, which weigh `weight` each.
struct Place {
  int tokens;
  double mass;
  unsigned int key;
  int rank;
  double weight;
};

// Where several parts add up a chunk's counters, the sums stay with the part that did
// (chunk top / 256 + i with part i mod kParts, 1 KiB each behind its Shared).
template <int kParts>
constexpr int kSumBytes = kParts >= 4 ? kChunks / kParts * 256 * 4 : 0;

// The search of one row, by one warp of CTA 0, descending from groups of 8 chunks to
// chunks, to 8 neighbouring keys and to a key, a lane for each. A warp alone runs at the
// pace at which its instructions are fetched, so all queries share this code.
template <int kParts>
struct Search {
  cg::cluster_group& cluster;
  Shared* sh;
  int lane;
  Scale scale;
  int group_n, group_t;   // tokens of chunks 8 lane .. 8 lane + 7, and of all before
  double group_m;         // their mass before

  // Tokens and mass before every chunk; returns the row's mass.
  __device__ __forceinline__ double prefixes() {
    group_n = 0;
    double m = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      group_n += sh->count[8 * lane + e];
      m += sh->mass[8 * lane + e];
    }
    group_t = warp_scan(group_n, lane) - group_n;
    const double through = warp_scan(m, lane), all = __shfl_sync(0xffffffffu, through, 31);
    group_m = lane == 0 ? 0.0 : through - m;
    int t = group_t;
    m = group_m;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sh->before[8 * lane + e] = t;
      sh->mass_before[8 * lane + e] = m;
      t += sh->count[8 * lane + e];
      m += sh->mass[8 * lane + e];
    }
    __syncwarp();
    return all;
  }

  // The last lane that has tokens and of whose first one the query holds; it always
  // holds of the first token of what is looked through (t == first_t).
  __device__ __forceinline__ int pick(const Query& query, bool some, int t, double m,
                                      int first_t) const {
    return 31 - __clz(__ballot_sync(0xffffffffu, some && (t == first_t || query.before(t, m))));
  }

  // The last token of which the query holds.
  __device__ __forceinline__ Place last(const Query& query) const {
    const int group = pick(query, group_n > 0, group_t, group_m, 0);
    // 8 chunks
    const int at = 8 * group + (lane & 7);
    int t = sh->before[at];
    double m = sh->mass_before[at];
    const int t0 = __shfl_sync(0xffffffffu, group_t, group);
    int from = pick(query, lane < 8 && sh->count[at] > 0, t, m, t0);
    const int chunk = 8 * group + from;
    const int t1 = __shfl_sync(0xffffffffu, t, from);
    const double m1 = __shfl_sync(0xffffffffu, m, from);
    // 32 times 8 keys
    unsigned int c[8];
    if (kParts >= 4) {
      const int i = chunk - static_cast<int>(scale.top >> 8);
      const uint4* sums = reinterpret_cast<const uint4*>(
          cluster.map_shared_rank(reinterpret_cast<uint32_t*>(sh + 1), i % kParts) +
          i / kParts * 256 + 8 * lane);
      const uint4 a = sums[0], b = sums[1];
      c[0] = a.x, c[1] = a.y, c[2] = a.z, c[3] = a.w;
      c[4] = b.x, c[5] = b.y, c[6] = b.z, c[7] = b.w;
    } else {
      counts8<kParts>(cluster, sh, 0, chunk * 32 + lane, c);
    }
    const unsigned int first = chunk * 256 + 8 * lane;
    const double ratio = scale.ratio(first);
    const Weights g = scale.from(first);
    double base = g.base;
    if (g.tiny) base = scale.exact(first);
    int n = 0;
    double x = 0.0;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      n += c[e];
      if (e >= g.shift) x = fma(x, ratio, as_double(c[e]));
    }
    x *= base;
    t = t1 + warp_scan(n, lane) - n;
    m = m1;
    {
      const double through = warp_scan(x, lane);
      if (lane > 0) m += through - x;
    }
    from = pick(query, n > 0, t, m, t1);
    // the 8 keys of that lane
    const int t2 = __shfl_sync(0xffffffffu, t, from);
    const double m2 = __shfl_sync(0xffffffffu, m, from);
    base = __shfl_sync(0xffffffffu, base, from);
    const int up = (lane & 7) - __shfl_sync(0xffffffffu, g.shift, from);
    n = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int v = __shfl_sync(0xffffffffu, static_cast<int>(c[e]), from);
      if (lane == e) n = v;
    }
    const double r2 = ratio * ratio;
    double w = up & 1 ? base * ratio : base;
    if (up & 2) w *= r2;
    if (up & 4) w *= r2 * r2;
    if (up < 0) w = 0.0;
    x = n * w;
    t = t2 + warp_scan(n, lane) - n;
    m = m2;
    {
      const double through = warp_scan(x, lane);
      if (lane > 0) m += through - x;
    }
    const int k = pick(query, n > 0, t, m, t2);
    n = __shfl_sync(0xffffffffu, n, k);
    t = __shfl_sync(0xffffffffu, t, k);
    m = __shfl_sync(0xffffffffu, m, k);
    w = __shfl_sync(0xffffffffu, w, k);
    const int r = query.within(t, m, w, n) - 1;
    return Place{t + r, m + r * w, static_cast<unsigned int>(chunk * 256 + 8 * from + k), r, w};
  }
};

template <int kParts>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared* sh = reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int part = static_cast<int>(cluster.block_rank());
  const int64_t r = blockIdx.x / kParts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const __half* row = p.logits + r * p.stride;
  const int lo = static_cast<int>(min(static_cast<int64_t>(part) * p.part,
                                      static_cast<int64_t>(p.vocab)));
  const int hi = min(lo + p.part, p.vocab);
  // tokens in front of the first 16-byte boundary, 16-byte units, tokens behind them
  const int head = min(static_cast<int>((-reinterpret_cast<intptr_t>(row + lo) & 15) >> 1), hi - lo);
  const int n8 = (hi - lo - head) >> 3, tail = (hi - lo - head) & 7;
  const __half* body = row + lo + head;
  const uint4* row8 = reinterpret_cast<const uint4*>(body);

  // ---- 1. histogram of this part ------------------------------------------------
  // the row's numbers, long before they are needed
  const float t32 = p.temperature[r], u32 = p.uniform[r];
  const float p32 = p.top_p ? p.top_p[r] : 1.f, m32 = p.min_p ? p.min_p[r] : 0.f;
  const int64_t k64 = p.top_k ? p.top_k[r] : 0;
  cluster.barrier_arrive();  // (this CTA runs: the others may write its shared memory)
  constexpr int kUnroll = 4;
  uint4 u[kUnroll];  // the first tokens are on their way while the counters are cleared
  auto fetch = [&](int i) {
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (i + k * kThreads < n8) u[k] = row8[i + k * kThreads];
  };
  fetch(threadIdx.x);
  for (int i = threadIdx.x; i < kKeys / 8; i += kThreads)
    reinterpret_cast<uint4*>(sh->hist)[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x < kChunks) {
    sh->count[threadIdx.x] = sh->above[threadIdx.x] = 0;
    sh->mass[threadIdx.x] = sh->mass_above[threadIdx.x] = 0.0;
  }
  if (threadIdx.x == 0) {
    sh->top = kKeys;
    sh->bottom = sh->some = 0;
  }
  __syncthreads();
  uint32_t top2 = 0xffffffffu, bottom2 = 0u;  // of even and odd tokens
  auto count = [&](unsigned int key) { atomicAdd(&sh->hist[key >> 1], (key & 1u) * 0xffffu + 1u); };
  auto count2 = [&](uint32_t bits) {
    const uint32_t k = keys_of2(bits);
    top2 = __vminu2(top2, k);
    bottom2 = __vmaxu2(bottom2, k);
    count(k & 0xffffu);
    count(k >> 16);
  };
  for (int i = threadIdx.x; i < n8; i += kUnroll * kThreads) {
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (i + k * kThreads >= n8) break;
      count2(u[k].x);
      count2(u[k].y);
      count2(u[k].z);
      count2(u[k].w);
    }
    fetch(i + kUnroll * kThreads);
  }
  if (threadIdx.x < head + tail) {
    const int i = threadIdx.x < head ? static_cast<int>(threadIdx.x) - head
                                     : 8 * n8 + static_cast<int>(threadIdx.x) - head;
    const uint32_t k = keys_of2(__half_as_ushort(body[i])) & 0xffffu;
    top2 = __vminu2(top2, 0xffff0000u | k);
    bottom2 = __vmaxu2(bottom2, k);
    count(k);
  }
  unsigned int top = __reduce_min_sync(0xffffffffu, min(top2 & 0xffffu, top2 >> 16));
  unsigned int bottom = __reduce_max_sync(0xffffffffu, max(bottom2 & 0xffffu, bottom2 >> 16));
  if (lane == 0) {
    atomicMin(&sh->top, top);
    atomicMax(&sh->bottom, bottom);
  }
  cluster.barrier_wait();
  __syncthreads();
  if (threadIdx.x == 0) {
    // -0 counts as +0; a part with a NaN says so with key 0 at its top
    sh->hist[kPlusZero >> 1] += (sh->hist[kMinusZero >> 1] & 0xffffu) << 16;
    sh->hist[kMinusZero >> 1] &= 0xffff0000u;
    if (sh->top == kMinusZero) sh->top = kPlusZero;
    if (sh->top < kPlusInf || sh->bottom > kMinusInf) sh->top = 0;
    for (int q = 0; q < kParts; ++q) {
      Shared* to = cluster.map_shared_rank(sh, q);
      to->tops[part] = sh->top;
      to->bottoms[part] = sh->bottom;
    }
  }
  cluster.sync();
  top = kKeys;
#pragma unroll
  for (int q = 0; q < kParts; ++q) {
    top = min(top, sh->tops[q]);
    bottom = max(bottom, sh->bottoms[q]);
  }

  const bool greedy = !(t32 > 0.f) || top == 0u || top >= kMinusInf;  // uniform over the cluster
  double step;
  const Scale scale{top, value_of(top, step), 1.0 / static_cast<double>(t32)};
  if (!greedy) {
    // ---- 2. tokens and mass of every chunk of keys that occur ---------------------
    const double min_p = static_cast<double>(m32);
    Shared* sh0 = cluster.map_shared_rank(sh, 0);
    // A lane sums up kGroup neighbouring keys, the lanes of a chunk together. Parts of a
    // row on SMs of their own have warps to spare and wait for each other's counters: 8
    // keys a lane there, a chunk a warp; 32 keys a lane, a binade a warp, else.
    constexpr int kGroup = kParts >= 4 ? 8 : 32, kLanes = 256 / kGroup;
#pragma unroll 1
    for (unsigned int unit = (top >> 8) / (kGroup / 8) + part + kParts * warp;
         unit <= (bottom >> 8) / (kGroup / 8); unit += kParts * (kThreads / 32)) {
      const unsigned int first = (unit * 32 + lane) * kGroup;
      const double ratio = scale.ratio(first), r2 = ratio * ratio, r4 = r2 * r2, r8 = r4 * r4;
      const Weights g = scale.from(first, kGroup);
      double base = g.base;
      if (g.tiny) base = scale.exact(first);
      const bool careful = m32 > 0.f || m32 != m32 || __any_sync(0xffffffffu, g.tiny);
      int n = 0, above = 0;
      double m = 0.0, ma = 0.0;
#pragma unroll
      for (int j = 0; j < kGroup / 8; ++j) {
        // lanes start at different eights: rows of 64 bytes otherwise share banks
        const int i = (j + (lane >> 1)) & (kGroup / 8 - 1);
        unsigned int c[8];
        counts8<kParts>(cluster, sh, part, static_cast<int>(first >> 3) + i, c);
        if (kParts >= 4) {
          uint4* sums = reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(sh + 1) +
                                                 (unit - (top >> 8)) / kParts * 256 + 8 * lane);
          sums[0] = make_uint4(c[0], c[1], c[2], c[3]);
          sums[1] = make_uint4(c[4], c[5], c[6], c[7]);
        }
        // x: weight of key 8 i of the group, then of the next keys
        double x = base;
        if (kGroup > 8) {
          const int up = max(8 * i - g.shift, 0);
          if (up & 1) x *= ratio;
          if (up & 2) x *= r2;
          if (up & 4) x *= r4;
          if (up & 8) x *= r8;
          if (up & 16) x *= r8 * r8;
        }
        if (!careful) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            n += c[e];
            m = fma(as_double(c[e]), x, m);
            if (8 * i + e >= g.shift) x *= ratio;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            n += c[e];
            const double y = as_double(c[e]) * x;
            m += y;
            if (x > 0.0 && x >= min_p) {
              above += c[e];
              ma += y;
            }
            if (8 * i + e >= g.shift) x *= ratio;
          }
        }
      }
      if (!careful) {
        above = n;
        ma = m;
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        m += __shfl_xor_sync(0xffffffffu, m, o);
        ma += __shfl_xor_sync(0xffffffffu, ma, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
        above += __shfl_xor_sync(0xffffffffu, above, o);
      }
      if (lane % kLanes == 0) {
        const int chunk = static_cast<int>(first >> 8);
        sh0->mass[chunk] = m;
        sh0->count[chunk] = n;
        sh0->mass_above[chunk] = ma;
        sh0->above[chunk] = above;
        if (above < n) sh0->some = 1;
      }
    }
    cluster.sync();
  }

  // ---- 3. the sampled token's key and rank ---------------------------------------
  if (part == 0 && warp == 0) {
    unsigned int key = top;
    int rank = 0;
    if (!greedy) {
      Search<kParts> s{cluster, sh, lane, scale};
      // kept: tokens of the shortest prefix so far, and its mass
      double all = s.prefixes(), mass = all;
      int kept = p.vocab;
      if (sh->some) {
        kept = 0;
        mass = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          kept += sh->above[32 * e + lane];
          mass += sh->mass_above[32 * e + lane];
        }
        kept = __reduce_add_sync(0xffffffffu, kept);
        mass = warp_sum(mass);
        if (kept == 0) {  // min_p above 1 keeps the first token all the same
          kept = 1;
          mass = 1.0;
        }
      }
      // the searches in turn: 0 the end of top-k, 1 the end of top-p, 2 the last token
      // with no more than u of the kept mass before it, 3 the last kept token when 2
      // comes out behind it
      Place z{};
      for (int turn = k64 > 0 && k64 < p.vocab ? 0 : p32 < 1.f ? 1 : 2; turn < 4;) {
        Query query{turn == 0 || turn == 3, turn == 2, turn == 0 ? static_cast<int>(k64) : kept,
                    turn == 1 ? static_cast<double>(p32) * all : static_cast<double>(u32) * mass};
        z = s.last(query);
        if (turn == 0) all = z.mass + z.weight;
        if (turn < 2 && z.tokens + 1 < kept) {
          kept = z.tokens + 1;
          mass = z.mass + z.weight;
        }
        turn = turn == 0 ? (p32 < 1.f ? 1 : 2) : turn == 1 ? 2 : turn == 2 && z.tokens >= kept ? 3 : 4;
      }
      key = z.key;
      rank = z.rank;
    }
    // tokens with that key before each part, to tell each its own rank (or that it has
    // none); of a row with a NaN the first part that has one looks
    int c = 0;
    if (lane < kParts) {
      if (key == 0) {
        c = sh->tops[lane] == 0;
      } else {
        const uint32_t w = *cluster.map_shared_rank(&sh->hist[key >> 1], lane);
        c = static_cast<int>((key & 1u) ? w >> 16 : w & 0xffffu);
      }
    }
    rank -= warp_scan(c, lane) - c;
    if (lane < kParts) {
      Shared* to = cluster.map_shared_rank(sh, lane);
      to->key = key;
      to->rank = rank < c ? rank : -1;
    }
  }
  cluster.sync();

  // ---- 4. its index: the rank-th token of this part with that key -------------------
  const unsigned int key = sh->key;
  int rank = sh->rank;
  if (rank < 0) return;
  // a tile of tokens in order, one group per thread: bit e of `hit` says that token
  // first + e of the row has the key. Counts the rank down; done below zero.
  auto tile = [&](unsigned int hit, int first) {
    const int n = __popc(hit), through = warp_scan(n, lane);
    __syncthreads();  // (the last tile's sums have been read)
    if (lane == 31) sh->warp_sum[warp] = through;
    __syncthreads();
    const int sum = lane < kThreads / 32 ? sh->warp_sum[lane] : 0;
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? sum : 0);
    const int here = rank - before - (through - n);
    if (here >= 0 && here < n) {
      for (int e = 0; e < here; ++e) hit &= hit - 1;
      p.out[r] = first + __ffs(hit) - 1;
    }
    rank -= __reduce_add_sync(0xffffffffu, sum);
  };
  auto is_key = [&](unsigned int bits) -> unsigned int { return key_of(bits & 0xffffu) == key; };
  fetch(threadIdx.x);
  if (head > 0)
    tile(threadIdx.x < head && is_key(__half_as_ushort(row[lo + threadIdx.x])), lo + threadIdx.x);
  for (int i0 = 0; i0 < n8 && rank >= 0; i0 += kUnroll * kThreads) {
    unsigned int hit[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      hit[k] = 0;
      if (i0 + k * kThreads + threadIdx.x < n8) {
        const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          hit[k] |= is_key(w[e]) << (2 * e) | is_key(w[e] >> 16) << (2 * e + 1);
      }
    }
    fetch(i0 + kUnroll * kThreads + threadIdx.x);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (rank >= 0 && i0 + k * kThreads < n8)
        tile(hit[k], lo + head + 8 * (i0 + k * kThreads + static_cast<int>(threadIdx.x)));
  }
  if (rank >= 0 && tail > 0) {
    const int i = 8 * n8 + static_cast<int>(threadIdx.x);
    tile(threadIdx.x < tail && is_key(__half_as_ushort(body[i])), lo + head + i);
  }
}

template <int kParts>
int launch(const Params& p, int64_t rows, int slot, cudaStream_t stream) {
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(&sample_kernel<kParts>),
                                       static_cast<int>(sizeof(Shared)) + kSumBytes<kParts>, slot);
  if (st != CIE_OK) return st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kParts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * kParts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared) + kSumBytes<kParts>;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<kParts>, p);
  if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
  return CIE_OK;
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (parts) {
    case 1: return launch<1>(p, rows, 5, st);
    case 2: return launch<2>(p, rows, 6, st);
    case 4: return launch<4>(p, rows, 7, st);
    default: return launch<8>(p, rows, 10, st);
  }
}

}  // extern "C"
