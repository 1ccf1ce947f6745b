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
//   1. every CTA counts its part into 2^16 16-bit counters in its shared memory (two to a
//      word, 128 KiB). A key that 4 of 32 sampled tokens have is counted in registers
//      instead: in a masked row most tokens are alike, and atomics on one address take
//      turns (64 rows of 151936, 99 % masked: 68 us without this, 23 us with it). Parts
//      of up to 98296 tokens save waves of CTAs (64 rows of 151936: 29 us as 4 parts a row,
//      21 us as 2); one key at most of such a part has 65536 tokens or more, and its
//      counter is kept less 65536 with the key noted;
//   2. the keys form 256 chunks of 8 entries of 32 keys (an entry lies in one binade, so its
//      weights are a geometric sequence); warps sum the counters over the cluster
//      (distributed shared memory) and hand CTA 0 each chunk's tokens, mass and tokens
//      that min-p keeps, and each entry's weight and what comes before it in its chunk;
//   3. CTA 0's first warp finds the kept prefix and the key of the sampled token
//      with its rank among the tokens of that key, descending to one entry's keys for
//      each prefix;
//   4. the CTA whose part holds that token looks it up in the row, whose first tokens were
//      loaded again during the search.
//
// Measured (B200, device time in a graph of calls): one row of 151936 14 us, 64 rows 21 us,
// 256 rows of 32003 27 us; with top-k, top-p and min-p 2 to 4 us more. What bounds it, of the 16 us of a CTA
// that counts 75968 tokens: shared atomics on random banks 6.5 us (6 tokens a cycle), the
// chunks' sums 4 us (fp64 latency, and distributed shared memory at about 22 bytes a cycle
// and SM), each search 1.7 us (one warp), clearing, barriers and look-up the rest. One CTA
// runs per SM, for two reasons: 126 to 128 registers x 512 threads are all that an SM has, and
// 181 KiB of shared memory (128 of them counters, 53 the searches' tables) more than half. So
// more than 148 CTAs take another wave: 256 rows of 151936, in clusters of two, 87 us.
// The clusters of eight spill 68 bytes.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "cie_host.h"
#include "cie_model_ops.h"

namespace cie {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kKeys = 1 << 16;
constexpr int kChunks = 256;              // of 8 entries
constexpr int kEntries = 8 * kChunks;     // of 32 keys
constexpr int kUnroll = 8;                // 16-byte units of the row in flight per thread
constexpr int kMaxPart = 98296;           // tokens of a part: multiple of 8 below 1.5 * 2^16
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 524224;
constexpr unsigned int kNone = 0xffffffffu;  // no key
constexpr int kOften = 4;  // of 32 sampled tokens: the key is counted apart
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

// Powers 1, 2, 4, 8 and 16 of the weight of a key by that of the one before.
struct Ratios {
  double r1, r2, r4, r8, r16;

  __device__ __forceinline__ double power(int n) const {  // 0 <= n < 32
    const double a = (n & 1 ? r1 : 1.0) * (n & 2 ? r2 : 1.0);
    const double b = (n & 4 ? r4 : 1.0) * (n & 8 ? r8 : 1.0);
    return n & 16 ? a * (b * r16) : a * b;
  }
};

struct alignas(16) Shared {
  uint32_t hist[kKeys / 2];       // counter of key d: half d & 1 of word d >> 1
  Ratios ratios[32];              // of each binade
  // CTA 0, per entry: weight of its first key (at or behind the row's largest logit), and
  // mass and tokens of the entries before it in its chunk
  double entry_base[kEntries], entry_mass[kEntries];
  // per chunk: mass and tokens, those of all chunks before, and those that min-p
  // keeps (`some` says that it drops any)
  double mass[kChunks], mass_before[kChunks], mass_above[kChunks];
  int entry_count[kEntries];
  int count[kChunks], before[kChunks], above[kChunks];
  int some;
  alignas(16) int hits[2][kUnroll * kThreads / 32];
  unsigned int top, bottom;       // smallest and largest key of this CTA's part
  unsigned int often;             // the key that is counted in registers
  unsigned int extra;             // the key whose counter lacks 65536
  int run, pairs;                 // tokens of key `often`; pairs of equal other ones
  // of every part
  unsigned int tops[kMaxCluster], bottoms[kMaxCluster], extras[kMaxCluster];
  unsigned int key;               // the sampled token's key and its rank among this
  int rank;                       // part's tokens of that key (negative: not here)
  int tokens;                     // how many those are
  int found;                      // tokens listed so far
  unsigned int unit;              // of chunk sums, the next one to take up
  int list[kThreads];
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
__device__ __forceinline__ int binade_of(unsigned int key) {
  return static_cast<int>((key >= 0x8000u ? key : 0x7fffu - key) >> 10 & 31u);
}
__device__ __forceinline__ double step_of(int binade) { return -exp2_of(max(binade, 1) - 25); }
__device__ __forceinline__ double value_of(unsigned int key, double& step) {
  const unsigned int bits = key >= 0x8000u ? key : 0x7fffu - key;
  const int binade = binade_of(key);
  const unsigned int whole = (bits & 1023u) + (binade ? 1024u : 0u);
  step = step_of(binade);
  return as_double(whole) * ((bits & 0x8000u) ? step : -step);
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
// if first lies above the row's largest logit. One exponential and the binade's ratio for
// 8 or 32 weights, each within 2^-47 of exp((value - peak) / temp).
struct Weights {
  double base;
  int shift;
  bool tiny;  // some of the keys may weigh 0: take base from Scale::exact
};

struct Scale {
  unsigned int top;      // the row's smallest key
  double peak, inv_temp; // its value, 1 / temperature

  // the weights of two neighbouring keys of a binade, one by the other, and its powers
  __device__ __forceinline__ Ratios ratios(int binade) const {
    const double x = step_of(binade) * inv_temp;
    Ratios r;
    r.r1 = x < -700.0 ? 0.0 : exp_above_700(fmin(fmax(x, -700.0), 0.0));
    r.r2 = r.r1 * r.r1;
    r.r4 = r.r2 * r.r2;
    r.r8 = r.r4 * r.r4;
    r.r16 = r.r8 * r.r8;
    return r;
  }

  __device__ __forceinline__ Weights from(unsigned int first, double keys) const {
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

// Counters of keys [8 j, 8 j + 8), of every part from part `first` on (each part begins with
// its own, so that no part is read by all at once) ...
template <int kParts>
__device__ __forceinline__ void load8(cg::cluster_group& cluster, Shared* sh, int first, int j,
                                      uint4 (&u)[kParts]) {
#pragma unroll
  for (int r = 0; r < kParts; ++r)
    u[r] = reinterpret_cast<const uint4*>(
        cluster.map_shared_rank(sh->hist, (first + r) % kParts))[j];
}
// ... and summed.
template <int kParts>
__device__ __forceinline__ void sum8(const uint4 (&u)[kParts], unsigned int (&c)[8]) {
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

// Adds the 65536 that a part's counter of one of the keys [first, first + 8) may lack.
template <int kParts>
__device__ __forceinline__ void add_extras(const Shared* sh, unsigned int first,
                                           unsigned int (&c)[8]) {
#pragma unroll 1
  for (int r = 0; r < kParts; ++r) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (sh->extras[r] == first + e) c[e] += 65536u;
  }
}

// c moved down by n places (0 <= n < 8), with zeros behind.
__device__ __forceinline__ void drop(unsigned int (&c)[8], int n) {
#pragma unroll
  for (int b = 1; b < 8; b <<= 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n & b) c[e] = e + b < 8 ? c[e + b] : 0u;
  }
}

// sum over e of c[e] * r^e, in a tree (a step of fp64 takes longer than the whole tree's issue)
__device__ __forceinline__ double weighted(const unsigned int (&c)[8], const Ratios& r) {
  const double a = fma(r.r1, as_double(c[1]), as_double(c[0]));
  const double b = fma(r.r1, as_double(c[3]), as_double(c[2]));
  const double d = fma(r.r1, as_double(c[5]), as_double(c[4]));
  const double e = fma(r.r1, as_double(c[7]), as_double(c[6]));
  return fma(r.r4, fma(r.r2, e, d), fma(r.r2, b, a));
}

// Inclusive sums over the lanes of each group of kLanes.
template <int kLanes = 32, typename T>
__device__ __forceinline__ T warp_scan(T v, int lane) {
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    const T x = __shfl_up_sync(0xffffffffu, v, o, kLanes);
    if (lane % kLanes >= o) v += x;
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
    if (c == 1) return 1;
    if (by_count) return max(1, min(count - t, c));
    const double q = (mass - m) / w;
    const double n = or_equal ? floor(q) + 1.0 : ceil(q);
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

// The search of one row, by one warp of CTA 0, descending from groups of 8 chunks to
// chunks, entries and keys, a lane for each. A warp alone runs at the pace at which its
// instructions are fetched, so all queries share this code.
template <int kParts>
struct Search {
  cg::cluster_group& cluster;
  Shared* sh;
  int lane;
  unsigned int top;
  bool extras;            // some counter lacks 65536
  int group_n, group_t;   // tokens of chunks 8 lane .. 8 lane + 7, and of all before
  double group_m;         // their mass before

  // Tokens and mass before every chunk; returns the row's mass.
  __device__ __forceinline__ double prefixes() {
    int n[8];
    double x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      n[e] = sh->count[8 * lane + e];
      x[e] = sh->mass[8 * lane + e];
    }
    const double s01 = x[0] + x[1], s23 = x[2] + x[3], s45 = x[4] + x[5], s67 = x[6] + x[7];
    const double s03 = s01 + s23, s05 = s03 + s45;
    const double in[8] = {0.0, x[0], s01, s01 + x[2], s03, s03 + x[4], s05, s05 + x[6]};
    const double through = warp_scan(s03 + (s45 + s67), lane);
    const double all = __shfl_sync(0xffffffffu, through, 31);
    const double m = __shfl_up_sync(0xffffffffu, through, 1);
    group_m = lane == 0 ? 0.0 : m;
    group_n = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) group_n += n[e];
    group_t = warp_scan(group_n, lane) - group_n;
    int t = group_t;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sh->before[8 * lane + e] = t;
      sh->mass_before[8 * lane + e] = group_m + in[e];
      t += n[e];
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
    // its 8 chunks
    const int at = 8 * group + (lane & 7);
    int n = sh->count[at], t = sh->before[at];
    double m = sh->mass_before[at];
    const int t0 = __shfl_sync(0xffffffffu, group_t, group);
    int from = pick(query, lane < 8 && n > 0, t, m, t0);
    const int chunk = 8 * group + from;
    const int t1 = __shfl_sync(0xffffffffu, t, from), through1 = t1 + __shfl_sync(0xffffffffu, n, from);
    const double m1 = __shfl_sync(0xffffffffu, m, from);
    // the chunk's 8 entries
    t = t1 + sh->entry_count[8 * chunk + (lane & 7)];
    m = m1 + sh->entry_mass[8 * chunk + (lane & 7)];
    const int behind = __shfl_down_sync(0xffffffffu, t, 1);
    from = pick(query, lane < 8 && (lane == 7 ? through1 : behind) > t, t, m, t1);
    const unsigned int entry = 8 * chunk + from;
    const int t2 = __shfl_sync(0xffffffffu, t, from);
    const double m2 = __shfl_sync(0xffffffffu, m, from);
    // the entry's 32 keys
    const unsigned int key = 32 * entry + lane;
    n = 0;
#pragma unroll
    for (int r = 0; r < kParts; ++r)
      n += reinterpret_cast<const unsigned short*>(cluster.map_shared_rank(sh->hist, r))[key];
    if (extras) {
#pragma unroll 1
      for (int r = 0; r < kParts; ++r) n += sh->extras[r] == key ? 65536 : 0;
    }
    const int up = static_cast<int>(key - max(32 * entry, top));
    double w = 0.0;
    if (up >= 0) w = sh->entry_base[entry] * sh->ratios[binade_of(key)].power(up);
    const double through = warp_scan(as_double(n) * w, lane);
    m = __shfl_up_sync(0xffffffffu, through, 1);
    m = lane == 0 ? m2 : m2 + m;
    t = t2 + warp_scan(n, lane) - n;
    from = pick(query, n > 0, t, m, t2);
    n = __shfl_sync(0xffffffffu, n, from);
    t = __shfl_sync(0xffffffffu, t, from);
    m = __shfl_sync(0xffffffffu, m, from);
    w = __shfl_sync(0xffffffffu, w, from);
    const int r = query.within(t, m, w, n) - 1;
    return Place{t + r, m + r * w, 32 * entry + from, r, w};
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
  // A programmatic dependent of the preceding kernel: the counters are cleared beside it, and
  // nothing of it is read or written before this waits (1.9 to 2.9 us a call).
  cluster.barrier_arrive();  // (this CTA runs: the others may write its shared memory)
  for (int i = threadIdx.x; i < kKeys / 8; i += kThreads)
    reinterpret_cast<uint4*>(sh->hist)[i] = make_uint4(0, 0, 0, 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint4 u[kUnroll];
  auto fetch = [&](int i) {
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (i + k * kThreads < n8) u[k] = row8[i + k * kThreads];
  };
  fetch(threadIdx.x);
  uint32_t sample = kNone;  // one of 32 tokens spread over the part
  if (warp == 0 && hi > lo)
    sample = __half_as_ushort(row[lo + static_cast<int>((hi - lo) * int64_t(lane) >> 5)]);
  // the row's numbers, long before they are needed
  const float t32 = p.temperature[r], u32 = p.uniform[r];
  const float p32 = p.top_p ? p.top_p[r] : 1.f, m32 = p.min_p ? p.min_p[r] : 0.f;
  const int64_t k64 = p.top_k ? p.top_k[r] : 0;
  if (threadIdx.x < kChunks) {
    sh->count[threadIdx.x] = sh->above[threadIdx.x] = 0;
    sh->mass[threadIdx.x] = sh->mass_above[threadIdx.x] = 0.0;
  }
  if (warp == 0) {
    const int times = __popc(__match_any_sync(0xffffffffu, sample));
    const int best = __reduce_max_sync(0xffffffffu, times << 5 | lane);
    uint32_t k = __shfl_sync(0xffffffffu, sample, best & 31);
    k = best >> 5 < kOften || k == kNone ? kNone : keys_of2(k) & 0xffffu;
    if (lane == 0) {
      sh->often = k;
      sh->extra = kNone;
      sh->top = kKeys;
      sh->bottom = sh->some = sh->run = sh->pairs = sh->found = 0;
      sh->unit = 0;
    }
  }
  __syncthreads();
  const unsigned int often = sh->often;
  int run = 0, pairs = 0;
  uint32_t top2 = 0xffffffffu, bottom2 = 0u;  // of even and odd tokens
  auto step_at = [](unsigned int key) { return (key & 1u) * 0xffffu + 1u; };
  // a comparison per token costs half of the loop's speed again: only where it pays
  auto count = [&](auto apart, unsigned int key) {
    if (decltype(apart)::value && key == often) ++run;
    else atomicAdd(&sh->hist[key >> 1], step_at(key));
  };
  auto count_all = [&](auto apart, auto wide) {
    auto count2 = [&](uint32_t bits) {
      const uint32_t k = keys_of2(bits);
      top2 = __vminu2(top2, k);
      bottom2 = __vmaxu2(bottom2, k);
      const unsigned int a = k & 0xffffu, b = k >> 16;
      if (decltype(wide)::value) pairs += a == b && !(decltype(apart)::value && b == often);
      count(apart, a);
      count(apart, b);
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
  };
  if (often != kNone) count_all(std::true_type{}, std::true_type{});
  else if (hi - lo > 65535) count_all(std::false_type{}, std::true_type{});
  else count_all(std::false_type{}, std::false_type{});
  if (threadIdx.x < head + tail) {
    const int i = threadIdx.x < head ? static_cast<int>(threadIdx.x) - head
                                     : 8 * n8 + static_cast<int>(threadIdx.x) - head;
    const uint32_t k = keys_of2(__half_as_ushort(body[i])) & 0xffffu;
    top2 = __vminu2(top2, 0xffff0000u | k);
    bottom2 = __vmaxu2(bottom2, k);
    count(std::true_type{}, k);
  }
  unsigned int top = __reduce_min_sync(0xffffffffu, min(top2 & 0xffffu, top2 >> 16));
  unsigned int bottom = __reduce_max_sync(0xffffffffu, max(bottom2 & 0xffffu, bottom2 >> 16));
  run = __reduce_add_sync(0xffffffffu, run);
  pairs = __reduce_add_sync(0xffffffffu, pairs);
  if (lane == 0) {
    atomicMin(&sh->top, top);
    atomicMax(&sh->bottom, bottom);
    atomicAdd(&sh->run, run);
    atomicAdd(&sh->pairs, pairs);
  }
  cluster.barrier_wait();
  __syncthreads();
  // 65536 tokens of one key among n fill at least 65536 - n / 2 of the part's pairs (16384
  // of the largest part's): only then can a counter have run over, and the part is counted
  // again with atomics that show it. (Two of a word never run over together.)
  const bool again = hi - lo > 65535 && sh->pairs >= 65536 - (hi - lo + 1) / 2 - 16;
  if (again) {
    for (int i = threadIdx.x; i < kKeys / 8; i += kThreads)
      reinterpret_cast<uint4*>(sh->hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i = lo + static_cast<int>(threadIdx.x); i < hi; i += kThreads) {
      const unsigned int k = keys_of2(__half_as_ushort(row[i])) & 0xffffu;
      const uint32_t old = atomicAdd(&sh->hist[k >> 1], step_at(k));
      if ((k & 1u ? old >> 16 : old & 0xffffu) == 0xffffu) {
        if (!(k & 1u)) atomicSub(&sh->hist[k >> 1], 0x10000u);  // the carry
        sh->extra = k;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    unsigned short* counters = reinterpret_cast<unsigned short*>(sh->hist);
    if (!again && often != kNone) {
      counters[often] = static_cast<unsigned short>(sh->run);
      if (sh->run >= 65536) sh->extra = often;
    }
    // -0 counts as +0; a part with a NaN says so with key 0 at its top
    const bool extra = sh->extra == kPlusZero || sh->extra == kMinusZero;
    const int zeros = counters[kPlusZero] + counters[kMinusZero] + (extra ? 65536 : 0);
    counters[kPlusZero] = static_cast<unsigned short>(zeros);
    counters[kMinusZero] = 0;
    if (zeros >= 65536) sh->extra = kPlusZero;
    else if (extra) sh->extra = kNone;
    if (sh->top == kMinusZero) sh->top = kPlusZero;
    if (sh->top < kPlusInf || sh->bottom > kMinusInf) sh->top = 0;
    for (int q = 0; q < kParts; ++q) {
      Shared* to = cluster.map_shared_rank(sh, q);
      to->tops[part] = sh->top;
      to->bottoms[part] = sh->bottom;
      to->extras[part] = sh->extra;
    }
  }
  const double inv_temp = 1.0 / static_cast<double>(t32);
  if (warp == 1) sh->ratios[lane] = Scale{0u, 0.0, inv_temp}.ratios(lane);
  cluster.sync();
  top = kKeys;
  bool extras = false;
#pragma unroll
  for (int q = 0; q < kParts; ++q) {
    extras |= sh->extras[q] != kNone;
    top = min(top, sh->tops[q]);
    bottom = max(bottom, sh->bottoms[q]);
  }

  const bool greedy = !(t32 > 0.f) || top == 0u || top >= kMinusInf;  // uniform over the cluster
  double step;
  const Scale scale{top, value_of(top, step), inv_temp};
  if (!greedy) {
    // ---- 2. tokens and mass of every chunk of keys that occur ---------------------
    const double min_p = static_cast<double>(m32);
    const bool filter = !(m32 <= 0.f);  // (a NaN keeps nothing but the first token)
    Shared* sh0 = cluster.map_shared_rank(sh, 0);
    // A lane sums up kGroup neighbouring keys, the lanes of a chunk together. Many parts
    // have warps to spare and wait for each other's counters: 8 keys a lane there, a chunk a
    // warp, the next chunk's counters on their way; 16 keys a lane in two parts, 32 (a binade
    // a warp) in one.
    constexpr bool kAhead = kParts >= 4;
    constexpr int kGroup = kParts == 1 ? 32 : kParts == 2 ? 16 : 8, kLanes = 256 / kGroup;
    constexpr int kWords = kGroup / 8;
    const unsigned int unit0 = (top >> 8) / kWords + part;
    const unsigned int units = (bottom >> 8) / kWords + 1;
    uint4 next[kWords][kParts];
    // lanes start at different eights: rows of 32 or 64 bytes otherwise share banks
    auto eight = [&](int j) { return (j + lane * kGroup / 64) & (kWords - 1); };
    auto load = [&](unsigned int unit) {
#pragma unroll
      for (int j = 0; j < kWords; ++j)
        load8<kParts>(cluster, sh, part, (unit * 32 + lane) * kWords + eight(j), next[j]);
    };
    // Empty units are soon done: warps take the next one when they are free.
    constexpr unsigned int kStep = kParts * (kThreads / 32);
    auto take = [&]() {
      const unsigned int n = lane == 0 ? atomicAdd(&sh->unit, 1u) : 0u;
      return unit0 + kParts * __shfl_sync(0xffffffffu, n, 0);
    };
    unsigned int unit = kAhead ? unit0 + kParts * warp : take();
    if (kAhead && unit < units) load(unit);
#pragma unroll 1
    for (; unit < units; unit = kAhead ? unit + kStep : take()) {
      const unsigned int first = (unit * 32 + lane) * kGroup;
      uint4 now[kWords][kParts];
      if (!kAhead) load(unit);
      uint32_t any = extras;
#pragma unroll
      for (int j = 0; j < kWords; ++j)
#pragma unroll
        for (int r = 0; r < kParts; ++r) {
          now[j][r] = next[j][r];
          any |= now[j][r].x | now[j][r].y | now[j][r].z | now[j][r].w;
        }
      if (kAhead && unit + kStep < units) load(unit + kStep);
      if (!__any_sync(0xffffffffu, any)) continue;  // (the binades next to zero)
      const Ratios ratios = sh->ratios[binade_of(first)];
      const Weights g = scale.from(first, kGroup);
      double base = g.base;
      if (g.tiny) base = scale.exact(first);
      // weights fall along a lane's keys: min-p keeps all of them, none, or (rarely) some
      const double least = base * (kGroup == 8 ? ratios.r8 : kGroup == 16 ? ratios.r16 : ratios.r16 * ratios.r16);
      const bool above_all = !filter || base >= min_p;
      const bool careful = __any_sync(
          0xffffffffu, g.tiny || (filter && base >= min_p && !(least > min_p * (1.0 + 1e-9))));
      const bool at_top = __any_sync(0xffffffffu, g.shift > 0);
      int n = 0, above = 0;
      double m = 0.0, ma = 0.0;
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const int i = eight(j);
        unsigned int c[8];
        sum8<kParts>(now[j], c);
        if (extras) add_extras<kParts>(sh, first + 8 * i, c);
        double x = base;  // weight of key 8 i of the group, or of the largest logit behind it
        if (kGroup > 8 && !at_top) x *= (i & 1 ? ratios.r8 : 1.0) * (i & 2 ? ratios.r16 : 1.0);
        if (at_top) {
          x *= ratios.power(max(8 * i - g.shift, 0));
          drop(c, min(max(g.shift - 8 * i, 0), 7));  // (no tokens above the largest logit)
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) n += c[e];
        if (!careful) {
          m = fma(weighted(c, ratios), x, m);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const double y = as_double(c[e]) * x;
            m += y;
            if (x > 0.0 && (!filter || x >= min_p)) {
              above += c[e];
              ma += y;
            }
            x *= ratios.r1;
          }
        }
      }
      if (!careful && above_all) {
        above = n;
        ma = m;
      }
      // what comes before each entry, and the chunk's sums
      const int through = warp_scan<kLanes>(n, lane);
      const double mass = warp_scan<kLanes>(m, lane);
      double before = __shfl_up_sync(0xffffffffu, mass, 1);
      if (lane % kLanes == 0) before = 0.0;
      if (lane % (32 / kGroup) == 0) {
        sh0->entry_base[first >> 5] = base;
        sh0->entry_mass[first >> 5] = before;
        sh0->entry_count[first >> 5] = through - n;
      }
      if (filter || careful) {
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) {
          ma += __shfl_xor_sync(0xffffffffu, ma, o);
          above += __shfl_xor_sync(0xffffffffu, above, o);
        }
      }
      if (lane % kLanes == kLanes - 1) {
        const int chunk = static_cast<int>(first >> 8);
        const bool all = !(filter || careful);
        sh0->mass[chunk] = mass;
        sh0->count[chunk] = through;
        sh0->mass_above[chunk] = all ? mass : ma;
        sh0->above[chunk] = all ? through : above;
        if (!all && above < through) sh0->some = 1;
      }
    }
    cluster.sync();
  }

  fetch(threadIdx.x);  // (for the look-up)
  // ---- 3. the sampled token's key and rank ---------------------------------------
  if (part == 0 && warp == 0) {
    unsigned int key = top;
    int rank = 0;
    if (!greedy) {
      Search<kParts> s{cluster, sh, lane, top, extras};
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
      const bool filter_p = !(p32 >= 1.f);  // (a NaN keeps nothing but the first token)
      for (int turn = k64 > 0 && k64 < p.vocab ? 0 : filter_p ? 1 : 2; turn < 4;) {
        Query query{turn == 0 || turn == 3, turn == 2, turn == 0 ? static_cast<int>(k64) : kept,
                    turn == 1 ? static_cast<double>(p32) * all : static_cast<double>(u32) * mass};
        z = s.last(query);
        if (turn == 0) all = z.mass + z.weight;
        if (turn < 2 && z.tokens + 1 < kept) {
          kept = z.tokens + 1;
          mass = z.mass + z.weight;
        }
        turn = turn == 0 ? (filter_p ? 1 : 2) : turn == 1 ? 2 : turn == 2 && z.tokens >= kept ? 3 : 4;
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
        c = static_cast<int>((key & 1u) ? w >> 16 : w & 0xffffu) +
            (sh->extras[lane] == key ? 65536 : 0);
      }
    }
    rank -= warp_scan(c, lane) - c;
    if (lane < kParts) {
      Shared* to = cluster.map_shared_rank(sh, lane);
      to->key = key;
      to->rank = rank < c ? rank : -1;
      to->tokens = c;
    }
  }
  cluster.sync();

  // ---- 4. its index: the rank-th token of this part with that key -------------------
  const unsigned int key = sh->key;
  int rank = sh->rank;
  if (rank < 0) return;
  if (key != 0 && sh->tokens <= kThreads) {
    // Few such tokens: listed in any order, then the one that has `rank` others before it.
    // Halves that differ from the key's bits in nothing (of a zero: nothing but the sign)
    // show up as the sign bit that x - 1 sets in a half x without one.
    const uint32_t mask = key == kPlusZero ? 0x7fff7fffu : 0xffffffffu;
    const uint32_t want = (key >= 0x8000u ? key : 0x7fffu - key) * 0x00010001u;
    auto miss = [&](uint32_t w) { return (w ^ want) & mask; };
    auto add = [&](int at) { sh->list[atomicAdd(&sh->found, 1)] = at; };
    for (int i = threadIdx.x; i < n8; i += kUnroll * kThreads) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        if (i + k * kThreads >= n8) break;
        const uint32_t x[4] = {miss(u[k].x), miss(u[k].y), miss(u[k].z), miss(u[k].w)};
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= (x[e] - 0x00010001u) & ~x[e];
        if (any & 0x80008000u) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((x[e >> 1] >> (e & 1) * 16 & 0xffffu) == 0) add(lo + head + 8 * (i + k * kThreads) + e);
        }
      }
      fetch(i + kUnroll * kThreads);
    }
    if (threadIdx.x < head + tail) {
      const int i = threadIdx.x < head ? static_cast<int>(threadIdx.x) - head
                                       : 8 * n8 + static_cast<int>(threadIdx.x) - head;
      if ((miss(__half_as_ushort(body[i])) & 0xffffu) == 0) add(lo + head + i);
    }
    __syncthreads();
    const int n = sh->tokens;
    if (static_cast<int>(threadIdx.x) < n) {
      const int at = sh->list[threadIdx.x];
      int before = 0;
      for (int i = 0; i < n; ++i) before += sh->list[i] < at;
      if (before == rank) p.out[r] = at;
    }
    return;
  }
  // kUnroll tiles of tokens in order, one group per thread and tile: bit e of hit[k] says
  // that token first + e of the row has the key, first = at + 8 (k kThreads + thread). Counts
  // the rank down; done below zero.
  int turn = 0;
  auto tiles = [&](const unsigned int (&hit)[kUnroll], int at, int width) {
    int* hits = sh->hits[turn & 1];  // (warps are at most one turn apart)
    ++turn;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int n = __reduce_add_sync(0xffffffffu, __popc(hit[k]));
      if (lane == 0) hits[k * (kThreads / 32) + warp] = n;
    }
    __syncthreads();
    static_assert(kUnroll * kThreads / 32 == 128, "four tiles of a warp per lane");
    const int4 four = reinterpret_cast<const int4*>(hits)[lane];
    const int sums[4] = {four.x, four.y, four.z, four.w};
    const int through = warp_scan(four.x + four.y + four.z + four.w, lane);
    const int all = __shfl_sync(0xffffffffu, through, 31);
    if (rank < all) {
      const int l = __ffs(__ballot_sync(0xffffffffu, through > rank)) - 1;
      int before = through - (four.x + four.y + four.z + four.w), which = 4 * lane;
#pragma unroll
      for (int e = 0; e < 3; ++e) {
        if (which == 4 * lane + e && rank >= before + sums[e]) {
          before += sums[e];
          ++which;
        }
      }
      before = __shfl_sync(0xffffffffu, before, l);
      which = __shfl_sync(0xffffffffu, which, l);
      if (which % (kThreads / 32) == warp) {
        const int k = which / (kThreads / 32);
        unsigned int h = 0;
#pragma unroll
        for (int q = 0; q < kUnroll; ++q)
          if (q == k) h = hit[q];
        const int n = __popc(h);
        const int here = rank - before - (warp_scan(n, lane) - n);
        if (here >= 0 && here < n) {
          for (int e = 0; e < here; ++e) h &= h - 1;
          p.out[r] = at + width * (k * kThreads + static_cast<int>(threadIdx.x)) + __ffs(h) - 1;
        }
      }
    }
    rank -= all;
  };
  auto is_key = [&](unsigned int bits) -> unsigned int { return key_of(bits & 0xffffu) == key; };
  if (head > 0) {
    const unsigned int hit[kUnroll] = {
        static_cast<int>(threadIdx.x) < head && is_key(__half_as_ushort(row[lo + threadIdx.x]))};
    tiles(hit, lo, 1);
  }
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
    tiles(hit, lo + head + 8 * i0, 8);
  }
  if (rank >= 0 && tail > 0) {
    const unsigned int hit[kUnroll] = {static_cast<int>(threadIdx.x) < tail &&
                                       is_key(__half_as_ushort(body[8 * n8 + threadIdx.x]))};
    tiles(hit, lo + head + 8 * n8, 1);
  }
}

// Launch of `rows` clusters of kParts CTAs, a programmatic dependent.
template <int kParts>
struct Launch {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};

  Launch(int64_t rows, cudaStream_t stream) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kParts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(rows * kParts));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }

  static int prepare() {
    constexpr int kSlot = kParts == 1 ? 5 : kParts == 2 ? 6 : kParts == 4 ? 7 : 10;
    return ensure_smem_attribute(reinterpret_cast<const void*>(&sample_kernel<kParts>),
                                 sizeof(Shared), kSlot);
  }

  // rows whose clusters run at the same time (asked once per device; SMs of a GPC that do
  // not make up a cluster stay idle: 148 SMs hold 15 clusters of 8, 33 of 4, 74 of 2)
  static int64_t at_once() {
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];  // 0: not yet asked
    const int dev = current_device();
    int n = dev >= 0 && dev < kDevices ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
      Launch l(1, nullptr);
      l.cfg.numAttrs = 1;
      if (prepare() != CIE_OK ||
          cudaOccupancyMaxActiveClusters(&n, sample_kernel<kParts>, &l.cfg) != cudaSuccess || n < 1)
        return 0;
      if (dev >= 0 && dev < kDevices) known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
  }

  static int run(const Params& p, int64_t rows, cudaStream_t stream) {
    const int st = prepare();
    if (st != CIE_OK) return st;
    Launch l(rows, stream);
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, sample_kernel<kParts>, p);
    if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
    return CIE_OK;
  }
};

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
  if (vocab > kMaxVocab)
    return fail(CIE_ERR_UNSUPPORTED, "vocab %lld > %d", (long long)vocab, kMaxVocab);
  if (stride < vocab) return fail(CIE_ERR_INVALID_ARGUMENT, "row stride < vocab");
  if ((reinterpret_cast<uintptr_t>(logits) & 1) != 0)
    return fail(CIE_ERR_ALIGNMENT, "logits must be 2-byte aligned");
  // Parts a row needs, and more while all clusters still run at the same time and a part is
  // long enough (151936 tokens, few rows: 18.0 us in 2 parts, 13.0 in 4, 12.0 in 8; 32003: 12.3
  // in 1, 10.8 in 2, 9.8 in 4, 10.6 in 8; 8000: 9.0, 9.3, 8.9 and 10.0; one cluster too
  // many doubles the time: 14.1 us for 33 rows in 4 parts, 24.4 for 34).
  int parts = 1;
  auto part_of = [&](int c) { return (vocab + 8LL * c - 1) / (8LL * c) * 8; };
  while (part_of(parts) > kMaxPart) parts *= 2;
  if (parts == 1 && part_of(1) > 8192 && rows <= Launch<2>::at_once()) parts = 2;
  if (parts == 2 && part_of(2) > 4096 && rows <= Launch<4>::at_once()) parts = 4;
  if (parts == 4 && part_of(4) > 16384 && rows <= Launch<8>::at_once()) parts = 8;
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
    case 1: return Launch<1>::run(p, rows, st);
    case 2: return Launch<2>::run(p, rows, st);
    case 4: return Launch<4>::run(p, rows, st);
    default: return Launch<8>::run(p, rows, st);
  }
}

}  // extern "C"
