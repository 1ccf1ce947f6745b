// KV pages in 8 bits: quantised as they are written (with or without the rotary
// embedding of q and k), and read back to fp16 pages.
//
// The scale of a (page, K or V, kv head) is a power of two 2^e, the smallest with
// max |x| <= 127 * 2^e over the page's rows so far, and a code is rint(x / 2^e).
// A page fills over many decode steps, so its scale can grow after rows were
// stored; with powers of two that is a shift of the older codes, and a value ends
// at most one final step off (half a step for the final rounding, and the halves
// of all earlier steps together are less than another), where re-rounding to
// arbitrary scales would add half a step for each growth. x / 2^e is exact in
// fp32 and code * 2^e in fp16, so every code follows from the values alone. A page
// that was filled elsewhere may come with any scale; it keeps it while new rows fit.
//
// All rows of a page that a call writes are quantised together, by one warp per
// (page, K or V, kv head): lane l holds chunk l mod 8 (8 of the 64 values) of
// rows l / 8, l / 8 + 4, ..., so a row is one 128-byte read and one 64-byte write.
#include "cie_common.cuh"
#include "cie_host.h"
#include "cie_kv_q8.h"

namespace cie {
namespace kvq8 {

constexpr int kD = 64;
constexpr int kPage = 16;
constexpr int kWarps = 8;
constexpr int kMaxExp = 9;    // 127 * 2^9 = 65024: code * scale stays finite in fp16
constexpr int kMinExp = -24;  // the smallest fp16 subnormal: code * scale is exact in fp16

struct Args {
  // rows from the fused QKV projection (rotary embedding) ...
  const __half* qkv;      // (T, (hq + 2 hkv) * D), row stride qkv_tok
  int64_t qkv_tok;
  const __half* cos;      // (T, D), row stride cs_tok
  const __half* sin;
  int64_t cs_tok;
  __half* q_out;          // (T, hq, D) contiguous
  // ... or K and V rows as they are
  const __half* k_new;
  const __half* v_new;
  int64_t k_tok, k_head, v_tok, v_head;
  int vec;                // all rows start on 16-byte boundaries
  int8_t* k_cache;        // (n_pages, hkv, page, D)
  int8_t* v_cache;
  float* scales;          // (n_pages, 2, hkv)
  int64_t page_stride, head_stride;
  const int64_t* lens;    // decode: per slot
  const int64_t* cu;      // mixed: (batch + 1)
  const int64_t* kv_lens; // mixed: per sequence
  const int64_t* slot_ids;
  BlockTable table;
  int64_t tokens;
  int batch, hq, hkv;
  int64_t n_pages, n_slots, bt_stride;
  int64_t row_pages;      // entries of a block-table row
};

// A block-table row holds at most the pool's pages: rows that lie further apart are rows of a
// wider table, whose other columns are not this one's.
__host__ __device__ inline int64_t row_pages(int64_t bt_stride, int64_t n_pages) {
  return bt_stride < n_pages ? bt_stride : n_pages;
}

// Launched as a programmatic dependent of the preceding kernel: nothing is read or written
// before that one is done, and the next such kernel may be scheduled meanwhile.
__device__ __forceinline__ void start_as_dependent() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void load8(const __half* p, int vec, float (&x)[8]) {
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(h[e]);
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __half2float(p[e]);
  }
}

// x * cos + rot * sin in fp32, products and sum rounded one by one (no fused
// multiply-add), so that the result is the same wherever it is computed.
__device__ __forceinline__ float rot1(float x, float rot, float c, float s) {
  return __fadd_rn(__fmul_rn(x, c), __fmul_rn(rot, s));
}

// The smallest e in [kMinExp, kMaxExp] with amax <= 127 * 2^e.
__device__ __forceinline__ int need_exp(float amax) {
  const int bits = __float_as_int(amax);
  const int ex = (bits >> 23) - 127;
  // amax = m * 2^ex, 1 <= m < 2: 127 * 2^(ex - 6) holds it up to m = 127 / 64
  const int e = (bits & 0x7fffff) <= 0x7e0000 ? ex - 6 : ex - 5;
  return min(max(e, kMinExp), kMaxExp);
}

// The update calls store powers of two from 2^-24 to 2^9, under which x * (1 / scale) and
// code * (old / new) are exact in fp32.
__device__ __forceinline__ bool is_pow2_scale(float s) {
  return (__float_as_int(s) & 0x7fffff) == 0 && s >= 5.9604645e-8f && s <= 512.f;
}

// x / scale rounded to the nearest whole number, ties to even, by its exact value; near: x / scale
// to within 2^-22 of it. The remainder of the whole number next to `near` is exact (it is a
// multiple of the last place of x or scale and at most about scale / 2), so that it shows
// on which side of a tie the quotient lies.
__device__ __forceinline__ float nearest(float x, float near, float scale) {
  if (fabsf(x) >= 127.f * scale) return copysignf(127.f, x);
  const float q = rintf(near), r = __fmaf_rn(-q, scale, x), half = 0.5f * scale;
  const bool odd = static_cast<int>(q) & 1;
  return fabsf(r) > half || (fabsf(r) == half && odd) ? q + copysignf(1.f, r) : q;
}

// Sequence of token t of a mixed pass: the first b with cu[b + 1] > t, or -1 when
// t lies in no sequence. `cu` is a.cu or a copy of it in shared memory.
__device__ __forceinline__ int find_seq(const int64_t* cu, int batch, int64_t t) {
  int lo = 0, hi = batch;  // cu[lo] <= t as far as cu is monotone
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo < batch && cu[lo] <= t ? lo : -1;
}

// Token t leads the rows that this call writes into one page when it is its
// sequence's first row or sits on row 0 of the page. Returns how many rows that
// is (0: t leads none, or must not be written), with the sequence and position.
template <bool kMixed>
__device__ __forceinline__ int led_rows(const Args& a, const int64_t* cu, int64_t t, int& b,
                                        int64_t& pos) {
  if (t >= a.tokens) return 0;
  if (!kMixed) {
    b = static_cast<int>(t);
    const int64_t slot = a.slot_ids[b];
    if (slot < 0 || slot >= a.n_slots) {
      raise_error(CIE_DEVERR_BAD_SLOT);
      return 0;
    }
    pos = a.lens[slot];
  } else {
    b = find_seq(cu, a.batch, t);
    if (b < 0) return 0;
    pos = a.kv_lens[b] + t - cu[b];
    if (t != cu[b] && (pos & (kPage - 1)) != 0) return 0;
  }
  if (pos < 0 || pos / kPage >= a.row_pages) {
    raise_error(CIE_DEVERR_BAD_LENGTH);
    return 0;
  }
  if (!kMixed) return 1;
  const int64_t left = min(cu[b + 1], a.tokens) - t;
  return static_cast<int>(min(left, static_cast<int64_t>(kPage - (pos & (kPage - 1)))));
}

// Whether a later sequence (with rows) writes the same slot: its rows win.
// Every lane of the warp takes part.
template <bool kMixed>
__device__ __forceinline__ bool superseded(const Args& a, int b, int64_t slot, int lane) {
  bool later = false;
  for (int i = b + 1 + lane; i < a.batch; i += 32)
    later |= a.slot_ids[i] == slot && (!kMixed || a.cu[i + 1] > a.cu[i]);
  return __any_sync(0xffffffffu, later);
}

// Quantises the n rows led by token t into their page: one warp, one of K / V,
// one kv head.
template <bool kRope, bool kMixed>
__device__ __forceinline__ void write_rows(const Args& a, int64_t t, int b, int64_t pos, int n,
                                           int which, int h, int lane) {
  const int64_t slot = a.slot_ids[b];
  if (slot < 0 || slot >= a.n_slots) {
    raise_error(CIE_DEVERR_BAD_SLOT);
    return;
  }
  const int64_t page = a.table.at(slot * a.bt_stride + pos / kPage);  // on its way
  const int off = static_cast<int>(pos & (kPage - 1));
  const int r = lane >> 3, c = lane & 7;

  float x[4][8];
  float amax = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + r;
    if (row < n) {
      const int64_t tok = t + row;
      if (kRope) {
        const __half* src = a.qkv + tok * a.qkv_tok + (a.hq + which * a.hkv + h) * kD;
        load8(src + 8 * c, 1, x[i]);
        if (which == 0) {
          float p[8], cs[8], sn[8];
          load8(src + 8 * (c ^ 4), 1, p);
          load8(a.cos + tok * a.cs_tok + 8 * c, 1, cs);
          load8(a.sin + tok * a.cs_tok + 8 * c, 1, sn);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] = rot1(x[i][e], c < 4 ? -p[e] : p[e], cs[e], sn[e]);
        }
      } else {
        load8(which ? a.v_new + tok * a.v_tok + h * a.v_head + 8 * c
                    : a.k_new + tok * a.k_tok + h * a.k_head + 8 * c,
              a.vec, x[i]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        finite = finite && fabsf(x[i][e]) <= 3.4028235e38f;
        if (x[i][e] != x[i][e]) x[i][e] = 0.f;
        amax = fmaxf(amax, fabsf(x[i][e]));
      }
    }
  }
  const bool skip = superseded<kMixed>(a, b, slot, lane);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (page < 0 || page >= a.n_pages) {
    raise_error(CIE_DEVERR_BAD_PAGE);
    return;
  }
  if (skip) return;
  if (!finite) raise_error(CIE_DEVERR_NONFINITE);

  float* sp = a.scales + page * 2 * a.hkv + which * a.hkv + h;
  int8_t* tile = (which ? a.v_cache : a.k_cache) + page * a.page_stride + h * a.head_stride;
  float stored = off > 0 ? *sp : 0.f;
  if (!(stored >= 0.f && stored <= 3.4028235e38f)) {  // no scale: the rows hold no values
    raise_error(CIE_DEVERR_BAD_SCALE);
    stored = 0.f;
  }
  const float scale = fmaxf(stored, __int_as_float((need_exp(amax) + 127) << 23));
  if (off > 0 && scale != stored) {
    // the page's older rows (0 .. off - 1) under the new scale, which is a power of two, so
    // that the ratio is exact; the product is too when the old scale was one
    const float ratio = __fdiv_rn(stored, scale);
    auto recode_all = [&](auto recode) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * i + r;
        if (row < off) {
          char4* d = reinterpret_cast<char4*>(tile + row * kD + 8 * c);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            char4 v = d[k];
            v.x = static_cast<signed char>(recode(v.x));
            v.y = static_cast<signed char>(recode(v.y));
            v.z = static_cast<signed char>(recode(v.z));
            v.w = static_cast<signed char>(recode(v.w));
            d[k] = v;
          }
        }
      }
    };
    if (is_pow2_scale(stored)) {
      recode_all([&](signed char q) { return __float2int_rn(q * ratio); });
    } else {
      recode_all([&](signed char q) { return __double2int_rn(q * static_cast<double>(ratio)); });
    }
  }
  float inv = __fdiv_rn(1.f, scale);
  if (!is_pow2_scale(scale)) {  // (outside the loop below: one branch instead of 32)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (4 * i + r < n) x[i][e] = nearest(x[i][e], __fmul_rn(x[i][e], inv), scale);
    }
    inv = 1.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + r;
    if (row < n) {
      int q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        q[e] = __float2int_rn(fminf(fmaxf(__fmul_rn(x[i][e], inv), -127.f), 127.f));
      uint2 u;
      u.x = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | q[3] << 24;
      u.y = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | q[7] << 24;
      *reinterpret_cast<uint2*>(tile + (off + row) * kD + 8 * c) = u;
    }
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0 && scale != stored) *sp = scale;
}

// The first CTAs take `tile` consecutive tokens each: warp 0 finds the leading ones, then
// the warps share out their (leader, K / V, kv head) units. With the rotary embedding the
// CTAs behind them rotate q, a thread per (token, head, chunk pair). What bounds a call is
// the chain of dependent loads (cu_seqlens -> length, slot -> block table -> scale), so
// a CTA gets few units and the two kinds of work run side by side.
// Measured (B200, device time, q rotated too): a decode step of 8 rows 4.0 us, of 256 5.3 us, a
// mixed pass of 2048 rows 6.2 us (with the read back 10.0 us; 21.9 us with one kind of CTA).
constexpr int kTile = 4;
constexpr int kCuShared = 512;  // cu_seqlens entries that are searched in shared memory

template <bool kRope, bool kMixed>
__global__ void __launch_bounds__(32 * kWarps) update_kernel(const Args a, int unit_ctas) {
  __shared__ int s_count;
  __shared__ int s_n[kTile], s_b[kTile];
  __shared__ int64_t s_t[kTile], s_pos[kTile];
  __shared__ int64_t s_cu[kMixed ? kCuShared : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  start_as_dependent();
  if (!kRope || static_cast<int>(blockIdx.x) < unit_ctas) {
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int per = 2 * a.hkv;
    if (!kMixed) {  // every token leads a page of its own
      for (int u = warp; u < kTile * per; u += kWarps) {
        const int w = u % per;
        int b = 0;
        int64_t pos = 0;
        if (led_rows<false>(a, nullptr, t0 + u / per, b, pos))
          write_rows<kRope, false>(a, t0 + u / per, b, pos, 1, w / a.hkv, w % a.hkv, lane);
      }
      return;
    }
    const int64_t* cu = a.cu;
    {
      if (blockIdx.x == 0) {
        // starts at 0 or later, never falls, ends inside the rows
        bool bad = threadIdx.x == 0 && (a.cu[0] < 0 || a.cu[a.batch] > a.tokens);
        for (int i = threadIdx.x; i < a.batch; i += blockDim.x) bad |= a.cu[i + 1] < a.cu[i];
        if (bad) raise_error(CIE_DEVERR_BAD_SEQLENS);
      }
      if (a.batch < kCuShared) {
        for (int i = threadIdx.x; i <= a.batch; i += blockDim.x) s_cu[i] = a.cu[i];
        cu = s_cu;
        __syncthreads();
      }
    }
    if (warp == 0) {
      int b = 0;
      int64_t pos = 0;
      const int n = lane < kTile ? led_rows<kMixed>(a, cu, t0 + lane, b, pos) : 0;
      const unsigned int leads = __ballot_sync(0xffffffffu, n > 0);
      if (n > 0) {
        const int i = __popc(leads & ((1u << lane) - 1u));
        s_n[i] = n;
        s_b[i] = b;
        s_t[i] = t0 + lane;
        s_pos[i] = pos;
      }
      if (lane == 0) s_count = __popc(leads);
    }
    __syncthreads();
    for (int u = warp; u < s_count * per; u += kWarps) {
      const int i = u / per, w = u % per;
      write_rows<kRope, kMixed>(a, s_t[i], s_b[i], s_pos[i], s_n[i], w / a.hkv, w % a.hkv, lane);
    }
    return;
  }
  // chunks c and c + 4 of a head are partners of the rotation
  const int64_t i = static_cast<int64_t>(blockIdx.x - unit_ctas) * blockDim.x + threadIdx.x;
  const int rows = a.hq * 4;
  const int64_t tok = i / rows;
  if (tok >= a.tokens) return;
  const int head = static_cast<int>(i - tok * rows) >> 2, c = static_cast<int>(i) & 3;
  const __half* src = a.qkv + tok * a.qkv_tok + head * kD + 8 * c;
  float x1[8], x2[8], c1[8], c2[8], s1[8], s2[8];
  load8(src, 1, x1);
  load8(src + 32, 1, x2);
  load8(a.cos + tok * a.cs_tok + 8 * c, 1, c1);
  load8(a.cos + tok * a.cs_tok + 32 + 8 * c, 1, c2);
  load8(a.sin + tok * a.cs_tok + 8 * c, 1, s1);
  load8(a.sin + tok * a.cs_tok + 32 + 8 * c, 1, s2);
  uint4 lo, hi;
  __half2* l = reinterpret_cast<__half2*>(&lo);
  __half2* g = reinterpret_cast<__half2*>(&hi);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int k = 2 * e;
    l[e] = __floats2half2_rn(rot1(x1[k], -x2[k], c1[k], s1[k]),
                             rot1(x1[k + 1], -x2[k + 1], c1[k + 1], s1[k + 1]));
    g[e] = __floats2half2_rn(rot1(x2[k], x1[k], c2[k], s2[k]),
                             rot1(x2[k + 1], x1[k + 1], c2[k + 1], s2[k + 1]));
  }
  __half* dst = a.q_out + (tok * a.hq + head) * kD + 8 * c;
  *reinterpret_cast<uint4*>(dst) = lo;
  *reinterpret_cast<uint4*>(dst + 32) = hi;
}

// ---- read back -------------------------------------------------------------------

struct ReadArgs {
  const int8_t* k;
  const int8_t* v;
  const float* scales;
  const int64_t* starts;  // may be null: all 0
  const int64_t* lens;
  const int64_t* slot_ids;
  BlockTable table;
  __half* k_out;
  __half* v_out;
  int hkv;
  int64_t n_pages, n_slots, bt_stride;
  int64_t page_stride, head_stride, out_page, out_head;
  int64_t row_pages;      // entries of a block-table row
};

// Two biased codes (code + 128) of `w`, picked by the selector, as fp16 numbers: 0x64 over a
// byte u is 1024 + u, and subtracting 1152 is exact.
__device__ __forceinline__ __half2 two_codes(uint32_t w, uint32_t sel) {
  const uint32_t h = __byte_perm(w, 0x64646464u, sel);
  return __hsub2(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(1152.f, 1152.f));
}

// 8 codes -> 8 fp16 values code * scale: rounded once, in fp16, when the scale is a fp16
// number (exact for the powers of two that the update calls store), else rounded to fp32
// and then to fp16.
__device__ __forceinline__ uint4 dequant8(uint2 codes, float scale) {
  const uint32_t w[2] = {codes.x ^ 0x80808080u, codes.y ^ 0x80808080u};
  const __half s = __float2half_rn(scale);
  const bool exact = __half2float(s) == scale;
  const __half2 s2 = __half2half2(s);
  uint4 r;
  __half2* o = reinterpret_cast<__half2*>(&r);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __half2 c = two_codes(w[e >> 1], e & 1 ? 0x4342 : 0x4140);
    if (exact) {
      o[e] = __hmul2_rn(c, s2);
    } else {
      const float2 f = __half22float2(c);
      o[e] = __floats2half2_rn(f.x * scale, f.y * scale);
    }
  }
  return r;
}

// Grid (x, sequence): a warp per K or V of a page, a lane per 8 codes (256-byte reads,
// 512-byte writes), two heads' reads in flight before their first write; a sequence's
// pages are dealt to its warps one by one. Bound by bandwidth, 1 byte read and 2 written
// a value: 32 x 8191 rows 19.0 us = 5.3 TB/s on a B200, 0.81 of a copy; 2047 rows 2.3 us.
// CTAs are dealt per sequence, absent ones too, so that one long history among them has few:
// 8191 rows alone 2.7 us, among 31 empty sequences 5.8 us, 63 8.9 us, 255 27 us.
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  start_as_dependent();
  const int64_t slot = a.slot_ids[b];
  int64_t len = a.lens[b], start = a.starts ? a.starts[b] : 0;
  if (slot < 0 || slot >= a.n_slots) {
    if (blockIdx.x == 0 && threadIdx.x == 0) raise_error(CIE_DEVERR_BAD_SLOT);
    return;
  }
  if (len > a.row_pages * kPage) {
    if (blockIdx.x == 0 && threadIdx.x == 0) raise_error(CIE_DEVERR_BAD_LENGTH);
    len = a.row_pages * kPage;
  }
  if (start < 0) start = 0;
  const int which = (threadIdx.x >> 5) & 1;
  const int8_t* pool = which ? a.v : a.k;
  __half* out = which ? a.v_out : a.k_out;
  const int64_t pages = (len + kPage - 1) / kPage;
  const int64_t* wide = static_cast<const int64_t*>(a.table.ptr);
  const int32_t* narrow = static_cast<const int32_t*>(a.table.ptr);
  const int64_t row = slot * a.bt_stride;
  auto entry = [&](int64_t j) -> int64_t {
    return j < pages ? (a.table.wide ? wide[row + j] : narrow[row + j]) : 0;
  };
  int64_t j = start / kPage + static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  int64_t page = entry(j);
#pragma unroll 1
  for (; j < pages;) {
    const int64_t next = j + static_cast<int64_t>(gridDim.x) * 4;
    const int64_t next_page = entry(next);
    if (page < 0 || page >= a.n_pages) {
      if (lane == 0) raise_error(CIE_DEVERR_BAD_PAGE);
    } else {
      const float* scales = a.scales + (page * 2 + which) * a.hkv;
      const int8_t* src = pool + page * a.page_stride + lane * 8;
      __half* dst = out + page * a.out_page + lane * 8;
      // rows lo .. hi - 1 of the page; chunk e of this lane is in row 4 e + lane / 8
      const int lo = static_cast<int>(max(start - j * kPage, int64_t(0))) - (lane >> 3);
      const int hi = static_cast<int>(min(len - j * kPage, int64_t(kPage))) - (lane >> 3);
#pragma unroll 1
      for (int h = 0; h < a.hkv; h += 2) {
        uint2 u[2][4];
        float s[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (h + k < a.hkv) {
            s[k] = scales[h + k];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              u[k][e] = *reinterpret_cast<const uint2*>(src + (h + k) * a.head_stride + 256 * e);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (h + k < a.hkv) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (4 * e >= lo && 4 * e < hi)
                *reinterpret_cast<uint4*>(dst + (h + k) * a.out_head + 256 * e) =
                    dequant8(u[k][e], s[k]);
          }
        }
      }
    }
    j = next;
    page = next_page;
  }
}

// ---- host side ---------------------------------------------------------------------

int check_pool(const void* k, const void* v, const void* scales, int hkv, int head_dim,
               int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
               int64_t page_stride, int64_t head_stride) {
  if (!k || !v || !scales) return fail(CIE_ERR_INVALID_ARGUMENT, "null pool or scales");
  if (head_dim != kD || page_size != kPage)
    return fail(CIE_ERR_UNSUPPORTED, "head_dim %d / page_size %d (supported: 64 / 16)", head_dim,
                page_size);
  if (hkv < 1 || hkv > 1024) return fail(CIE_ERR_UNSUPPORTED, "num_kv_heads %d", hkv);
  if (n_pages < 1 || n_slots < 1 || bt_stride < 1)
    return fail(CIE_ERR_INVALID_ARGUMENT, "n_pages / n_slots / bt_stride must be >= 1");
  if (head_stride < kPage * kD || page_stride < head_stride * hkv)
    return fail(CIE_ERR_INVALID_ARGUMENT, "overlapping pool strides (page %lld, head %lld)",
                (long long)page_stride, (long long)head_stride);
  if ((page_stride % 16) || (head_stride % 16) || !aligned16(k) || !aligned16(v) ||
      (reinterpret_cast<uintptr_t>(scales) & 3))
    return fail(CIE_ERR_ALIGNMENT, "pools must be 16-byte aligned with 16-byte strides, scales 4");
  return CIE_OK;
}

// Launch as a programmatic dependent (start_as_dependent).
template <typename Kernel, typename... Params>
int launch(const char* what, Kernel kernel, dim3 grid, cie_stream_t stream, Params... params) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params...);
  if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return CIE_OK;
}

template <bool kRope, bool kMixed>
int launch_update(const Args& a, cie_stream_t stream) {
  const int64_t units = (a.tokens + kTile - 1) / kTile;
  const int64_t rotate = kRope ? (a.tokens * a.hq * 4 + 32 * kWarps - 1) / (32 * kWarps) : 0;
  if (units + rotate > 0x7fffffff) return fail(CIE_ERR_OVERFLOW, "too many tokens");
  return launch("kv_q8 update", update_kernel<kRope, kMixed>,
                dim3(static_cast<unsigned>(units + rotate)), stream, a, static_cast<int>(units));
}

// Checks and launch of every update entry point: mixed when a.cu is set, with the
// rotary embedding when a.qkv is set.
int update(Args a, bool rope, bool mixed, int head_dim, int page_size, cie_stream_t stream) {
  if (a.batch < 0 || a.tokens < 0) return fail(CIE_ERR_INVALID_ARGUMENT, "negative batch / tokens");
  if (a.tokens == 0 || (a.batch == 0 && !rope)) return CIE_OK;
  const int st = check_pool(a.k_cache, a.v_cache, a.scales, a.hkv, head_dim, page_size, a.n_pages,
                            a.n_slots, a.bt_stride, a.page_stride, a.head_stride);
  if (st != CIE_OK) return st;
  if ((mixed && !a.cu) ||
      (a.batch > 0 && (!a.slot_ids || !a.table.ptr || (mixed ? !a.kv_lens : !a.lens))))
    return fail(CIE_ERR_INVALID_ARGUMENT, "null lengths / slot_ids / block_table");
  if (rope) {
    if (!a.qkv || !a.cos || !a.sin || !a.q_out)
      return fail(CIE_ERR_INVALID_ARGUMENT, "null qkv / cos / sin / q_out");
    if (a.hq < 1) return fail(CIE_ERR_INVALID_ARGUMENT, "num_q_heads must be >= 1");
    if (a.qkv_tok < static_cast<int64_t>(a.hq + 2 * a.hkv) * kD || a.cs_tok < kD)
      return fail(CIE_ERR_INVALID_ARGUMENT, "qkv / cos / sin rows overlap");
    if ((a.qkv_tok % 8) || (a.cs_tok % 8) || !aligned16(a.qkv) || !aligned16(a.cos) ||
        !aligned16(a.sin) || !aligned16(a.q_out))
      return fail(CIE_ERR_ALIGNMENT, "qkv / cos / sin / q_out rows must be 16-byte aligned");
    return mixed ? launch_update<true, true>(a, stream) : launch_update<true, false>(a, stream);
  }
  if (!a.k_new || !a.v_new) return fail(CIE_ERR_INVALID_ARGUMENT, "null k_new / v_new");
  a.vec = aligned16(a.k_new) && aligned16(a.v_new) && a.k_tok % 8 == 0 && a.k_head % 8 == 0 &&
          a.v_tok % 8 == 0 && a.v_head % 8 == 0;
  return mixed ? launch_update<false, true>(a, stream) : launch_update<false, false>(a, stream);
}

int read(const ReadArgs& a, int batch, int head_dim, int page_size, cie_stream_t stream) {
  if (batch < 0) return fail(CIE_ERR_INVALID_ARGUMENT, "batch < 0");
  if (batch == 0) return CIE_OK;
  const int st = check_pool(a.k, a.v, a.scales, a.hkv, head_dim, page_size, a.n_pages, a.n_slots,
                            a.bt_stride, a.page_stride, a.head_stride);
  if (st != CIE_OK) return st;
  if (!a.lens || !a.slot_ids || !a.table.ptr || !a.k_out || !a.v_out)
    return fail(CIE_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (batch > 65535) return fail(CIE_ERR_UNSUPPORTED, "batch %d > 65535", batch);
  if (a.out_head < kPage * kD || a.out_page < a.out_head * a.hkv)
    return fail(CIE_ERR_INVALID_ARGUMENT, "overlapping output strides");
  if ((a.out_page % 8) || (a.out_head % 8) || !aligned16(a.k_out) || !aligned16(a.v_out))
    return fail(CIE_ERR_ALIGNMENT, "outputs must be 16-byte aligned with 16-byte strides");
  // lengths are on the device: as many CTAs as the SMs hold, at most one per four pages of
  // the block-table row
  int64_t per = (8LL * sm_count() + batch - 1) / batch;
  if (per > (a.row_pages + 3) / 4) per = (a.row_pages + 3) / 4;
  return launch("kv_q8 read", read_kernel, dim3(static_cast<unsigned>(per), batch), stream, a);
}

Args pool_args(void* k_cache, void* v_cache, float* scales, const int64_t* slot_ids,
               BlockTable table, int batch, int hkv, int64_t n_pages, int64_t n_slots,
               int64_t bt_stride, int64_t page_stride, int64_t head_stride) {
  Args a{};
  a.k_cache = static_cast<int8_t*>(k_cache);
  a.v_cache = static_cast<int8_t*>(v_cache);
  a.scales = scales;
  a.slot_ids = slot_ids;
  a.table = table;
  a.batch = batch;
  a.hkv = hkv;
  a.n_pages = n_pages;
  a.n_slots = n_slots;
  a.bt_stride = bt_stride;
  a.row_pages = row_pages(bt_stride, n_pages);
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  return a;
}

void set_rows(Args& a, const void* k_new, const void* v_new, int64_t k_tok, int64_t k_head,
              int64_t v_tok, int64_t v_head) {
  a.k_new = static_cast<const __half*>(k_new);
  a.v_new = static_cast<const __half*>(v_new);
  a.k_tok = k_tok;
  a.k_head = k_head;
  a.v_tok = v_tok;
  a.v_head = v_head;
}

void set_rope(Args& a, const void* qkv, int64_t qkv_tok, const void* cos, const void* sin,
              int64_t cs_tok, void* q_out, int hq) {
  a.qkv = static_cast<const __half*>(qkv);
  a.qkv_tok = qkv_tok;
  a.cos = static_cast<const __half*>(cos);
  a.sin = static_cast<const __half*>(sin);
  a.cs_tok = cs_tok;
  a.q_out = static_cast<__half*>(q_out);
  a.hq = hq;
}

}  // namespace kvq8
}  // namespace cie

extern "C" {

int cie_kv_q8_decode_update(void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
    const int64_t* slot_ids, const int64_t* block_table, const void* k_new, const void* v_new,
    int batch, int num_kv_heads, int head_dim, int page_size, int64_t n_pages, int64_t n_slots,
    int64_t bt_stride, int64_t cache_page_stride, int64_t cache_head_stride,
    int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
    cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 1}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rows(a, k_new, v_new, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride);
  a.lens = lens;
  a.tokens = batch;
  return update(a, false, false, head_dim, page_size, stream);
}

int cie_kv_q8_mixed_update(void* k_cache, void* v_cache, float* kv_scales,
    const int64_t* cu_seqlens, const int64_t* kv_lens, const int64_t* slot_ids,
    const int64_t* block_table, const void* k_new, const void* v_new, int batch,
    int64_t num_tokens, int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
    int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride, int64_t cache_head_stride,
    int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
    cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 1}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rows(a, k_new, v_new, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride);
  a.cu = cu_seqlens;
  a.kv_lens = kv_lens;
  a.tokens = num_tokens;
  return update(a, false, true, head_dim, page_size, stream);
}

int cie_rope_kv_q8_decode_update(const void* qkv, int64_t qkv_tok_stride, const void* cos,
    const void* sin, int64_t cs_tok_stride, void* q_out, void* k_cache, void* v_cache,
    float* kv_scales, const int64_t* lens, const int64_t* slot_ids,
    const int64_t* block_table, int batch, int num_q_heads, int num_kv_heads, int head_dim,
    int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 1}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rope(a, qkv, qkv_tok_stride, cos, sin, cs_tok_stride, q_out, num_q_heads);
  a.lens = lens;
  a.tokens = batch;
  return update(a, true, false, head_dim, page_size, stream);
}

int cie_rope_kv_q8_mixed_update(const void* qkv, int64_t qkv_tok_stride, const void* cos,
    const void* sin, int64_t cs_tok_stride, void* q_out, void* k_cache, void* v_cache,
    float* kv_scales, const int64_t* cu_seqlens, const int64_t* kv_lens,
    const int64_t* slot_ids, const int64_t* block_table, int batch, int64_t num_tokens,
    int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
    int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride, int64_t cache_head_stride,
    cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 1}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rope(a, qkv, qkv_tok_stride, cos, sin, cs_tok_stride, q_out, num_q_heads);
  a.cu = cu_seqlens;
  a.kv_lens = kv_lens;
  a.tokens = num_tokens;
  return update(a, true, true, head_dim, page_size, stream);
}

int cie_kv_q8_read(const void* k_cache, const void* v_cache, const float* kv_scales,
    const int64_t* starts, const int64_t* lens, const int64_t* slot_ids,
    const int64_t* block_table, void* k_out, void* v_out, int batch, int num_kv_heads,
    int head_dim, int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, int64_t out_page_stride,
    int64_t out_head_stride, cie_stream_t stream) {
  const cie::kvq8::ReadArgs a{static_cast<const int8_t*>(k_cache),
                              static_cast<const int8_t*>(v_cache), kv_scales, starts, lens,
                              slot_ids, cie::BlockTable{block_table, 1},
                              static_cast<__half*>(k_out), static_cast<__half*>(v_out),
                              num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                              cache_head_stride, out_page_stride, out_head_stride,
                              cie::kvq8::row_pages(bt_stride, n_pages)};
  return cie::kvq8::read(a, batch, head_dim, page_size, stream);
}

int cie_kv_q8_decode_update_bt32(void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
    const int64_t* slot_ids, const int32_t* block_table, const void* k_new, const void* v_new,
    int batch, int num_kv_heads, int head_dim, int page_size, int64_t n_pages, int64_t n_slots,
    int64_t bt_stride, int64_t cache_page_stride, int64_t cache_head_stride,
    int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
    cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 0}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rows(a, k_new, v_new, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride);
  a.lens = lens;
  a.tokens = batch;
  return update(a, false, false, head_dim, page_size, stream);
}

int cie_kv_q8_mixed_update_bt32(void* k_cache, void* v_cache, float* kv_scales,
    const int64_t* cu_seqlens, const int64_t* kv_lens, const int64_t* slot_ids,
    const int32_t* block_table, const void* k_new, const void* v_new, int batch,
    int64_t num_tokens, int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
    int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride, int64_t cache_head_stride,
    int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
    cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 0}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rows(a, k_new, v_new, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride);
  a.cu = cu_seqlens;
  a.kv_lens = kv_lens;
  a.tokens = num_tokens;
  return update(a, false, true, head_dim, page_size, stream);
}

int cie_rope_kv_q8_decode_update_bt32(const void* qkv, int64_t qkv_tok_stride, const void* cos,
    const void* sin, int64_t cs_tok_stride, void* q_out, void* k_cache, void* v_cache,
    float* kv_scales, const int64_t* lens, const int64_t* slot_ids,
    const int32_t* block_table, int batch, int num_q_heads, int num_kv_heads, int head_dim,
    int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 0}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rope(a, qkv, qkv_tok_stride, cos, sin, cs_tok_stride, q_out, num_q_heads);
  a.lens = lens;
  a.tokens = batch;
  return update(a, true, false, head_dim, page_size, stream);
}

int cie_rope_kv_q8_mixed_update_bt32(const void* qkv, int64_t qkv_tok_stride, const void* cos,
    const void* sin, int64_t cs_tok_stride, void* q_out, void* k_cache, void* v_cache,
    float* kv_scales, const int64_t* cu_seqlens, const int64_t* kv_lens,
    const int64_t* slot_ids, const int32_t* block_table, int batch, int64_t num_tokens,
    int num_q_heads, int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
    int64_t n_slots, int64_t bt_stride, int64_t cache_page_stride, int64_t cache_head_stride,
    cie_stream_t stream) {
  using namespace cie::kvq8;
  Args a = pool_args(k_cache, v_cache, kv_scales, slot_ids, cie::BlockTable{block_table, 0}, batch,
                     num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                     cache_head_stride);
  set_rope(a, qkv, qkv_tok_stride, cos, sin, cs_tok_stride, q_out, num_q_heads);
  a.cu = cu_seqlens;
  a.kv_lens = kv_lens;
  a.tokens = num_tokens;
  return update(a, true, true, head_dim, page_size, stream);
}

int cie_kv_q8_read_bt32(const void* k_cache, const void* v_cache, const float* kv_scales,
    const int64_t* starts, const int64_t* lens, const int64_t* slot_ids,
    const int32_t* block_table, void* k_out, void* v_out, int batch, int num_kv_heads,
    int head_dim, int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, int64_t out_page_stride,
    int64_t out_head_stride, cie_stream_t stream) {
  const cie::kvq8::ReadArgs a{static_cast<const int8_t*>(k_cache),
                              static_cast<const int8_t*>(v_cache), kv_scales, starts, lens,
                              slot_ids, cie::BlockTable{block_table, 0},
                              static_cast<__half*>(k_out), static_cast<__half*>(v_out),
                              num_kv_heads, n_pages, n_slots, bt_stride, cache_page_stride,
                              cache_head_stride, out_page_stride, out_head_stride,
                              cie::kvq8::row_pages(bt_stride, n_pages)};
  return cie::kvq8::read(a, batch, head_dim, page_size, stream);
}

}  // extern "C"
