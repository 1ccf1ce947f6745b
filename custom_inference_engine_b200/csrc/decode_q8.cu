// Split-KV paged GQA decode attention over 8-bit pages (sm_100a).
//
// Mathematics, per page and kv head (16 keys, up to 8 query heads on the MMA's N
// side), warp-level MMA with fp16 operands and fp32 accumulation:
//   S^T (16 x 8) = Kc (16 x 64) . Q^T (64 x 8),  s = S^T * scale_k / 8
//   online softmax over keys in fp32; p = exp(s - m), rounded to fp16
//   O^T (64 x 8) = alpha O^T + scale_v * (Vc^T (64 x 16) . P^T (16 x 8))
// Codes are whole numbers up to 127, exact in fp16: a byte c + 128 under the
// exponent byte 0x64 is the fp16 number 1024 + 128 + c, and subtracting 1152 is
// exact. scale_k and scale_v multiply fp32 results, so neither p nor a code is
// ever scaled in fp16, whatever range the page scales span. p has the 11 bits of the MMA's
// operand: a second MMA on its remainder would double the P V products for an error that is
// the output's own rounding already (against 64 bits, as a share of the norm: 2.2e-4 to 2.5e-4,
// with 32-bit probabilities 1.9e-4 to 2.3e-4). Its sum l is of the fp32 values.
//
// Contraction indices and output rows may be numbered freely as long as both
// operands agree, so every lane's operand bytes are contiguous in memory and the two
// orders of a page's 16 rows keep shared-memory banks apart:
//   S: lane (g, t) takes bytes [16 t, 16 t + 16) of rows pi(g) and pi(g) + 8;
//      MMA step ks contracts dims 16 t + 4 ks + {0, 1, 2, 3}
//   O: lane (g, t) takes bytes [8 g, 8 g + 8) of rows pi(2t), pi(2t + 1), pi(2t) + 8 and
//      pi(2t + 1) + 8, which are MMA keys 2t, 2t + 1, 2t + 8, 2t + 9; MMA row g of tile mt
//      is dim 8 g + 2 mt, row g + 8 is dim 8 g + 2 mt + 1
// with pi(2 t) = t, pi(2 t + 1) = 4 + (t xor 1).
//
// Every warp brings its own pages into its own ring of shared memory (cp.async.bulk, one
// lane issues): half the bytes a page means twice the pages a second, and one thread
// that issued the copies of a whole CTA would bound it (a single issuer of 4 KiB copies
// streams about 30 GB/s).
//
// Work split: one CTA per (sequence, split), eight warps, each with two kv heads (or the
// only one) of every 8th page of the split (every 4th where there are four heads). Two
// heads a warp because their K tiles lie side by side, and so do their V tiles: with 16
// warps per SM, scattered reads of 1 KiB stream 5.1 TB/s and of 2 KiB 6.1 TB/s on a B200.
// The warps' results are merged in shared memory, those of several splits by a second
// kernel.
//
// Measured (B200, cold pages, a chain of calls in a graph, where a call's start overlaps the
// one before): 256 x 4096 rows, two heads, 52 us = 5.2 TB/s, 0.80 of the measured copy
// bandwidth; 64 x 16001-32768 83 us; one sequence of 511 rows 4.5 us, of 16384 7.4 us. Calls
// between events take 4 to 5 us more (56, 87 and 9.7 us for the first three). What bounds it:
// the pages' bandwidth at large sizes, with 16 warps per SM
// (128 registers) and about 240 instructions a page and head; the chain slot -> length ->
// block table -> page -> merge at small ones.
#include "cie_common.cuh"
#include "cie_host.h"
#include "cie_kv_q8.h"

namespace cie {
namespace dq8 {

constexpr int kD = 64;
constexpr int kPage = 16;
constexpr int kWarps = 8;
constexpr int kMaxGroup = 8;
constexpr int kTileBytes = 2 * kPage * kD;  // K and V of one page and kv head
constexpr int kAccStride = kD + 4;          // floats of one head in the merge buffer (banks)

template <int HKV>
struct Cfg {
  static constexpr int kHeads = HKV == 1 ? 1 : 2;       // kv heads per warp
  static constexpr int kStep = kWarps / (HKV / kHeads); // warps per page: pages apart
  static constexpr int kRing = HKV == 1 ? 4 : 2;  // pages in flight per warp
  static constexpr int kPageBytes = kHeads * kTileBytes;
  static constexpr int kBarOffset = kWarps * kRing * kPageBytes;
  static constexpr int kSmemBytes = kBarOffset + kWarps * kRing * 8;
  static_assert(kRing * kPageBytes >= kHeads * kMaxGroup * kAccStride * 4,
                "a warp's accumulators fit its ring");
};

struct Params {
  const __half* q;          // (B, H_q, D)
  const int8_t* k;          // (n_pages, HKV, 16, 64)
  const int8_t* v;
  const float* scales;      // (n_pages, 2, HKV)
  const int64_t* lens;      // (B,) keys; after an update of the call (n_slots,) without the new row
  const int64_t* slot_ids;  // (B,)
  BlockTable table;         // n_slots rows, bt_stride apart
  __half* o;                // (B, H_q, D)
  float* ws_acc;            // (B, S, H_q, D)
  float* ws_ml;             // (B, S, H_q, 2)
  int num_splits;
  int group;                // query heads per kv head, 1..8
  int after_update;         // q and each row's last page are the preceding kernel's
  int64_t n_pages, n_slots, bt_stride;
  int64_t row_pages;        // entries of a block-table row
  int64_t page_stride, head_stride;
};

// `bytes` contiguous bytes from global to shared memory, counted on mbarrier `bar`.
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(addr)
               : "memory");
  return r;
}

// D = A(16x16, row) * B(16x8, col), fp16 inputs, fp32 accumulate.
__device__ __forceinline__ void mma_16816_zero(float (&d)[4], uint32_t a0, uint32_t a1,
                                               uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Two biased codes of `w` (code + 128, picked by the selector) as a pair of fp16; high:
// 0x64 in every byte. It is passed in a register of its own (below): a constant that the
// compiler may keep in a uniform register is moved from there before every use, 28
// moves per page and head of 265 instructions.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w, uint32_t sel, uint32_t high) {
  uint32_t h = __byte_perm(w, high, sel);
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&h), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ int seq_pages(const Params& p, int b) {
  return decode::seq_pages(p.lens, p.slot_ids, b, p.n_slots, p.row_pages, p.after_update);
}

// kAfterUpdate: the preceding kernel is the same call's update, which writes q and, of
// every row's pages, the last one, with its scale. It has itself waited for everything before
// it when this grid starts, so that a warp's first pages are fetched while it runs (64 rows
// of 325 to 975 keys: 12.9 us for the call, 14.0 us as two calls; 256 of 1000 to 3000: 42.1 and
// 45.8). With two heads it spills 4 bytes at the cap of 128 registers.
// Rotating q here as well and waiting only before the last page is read won 0.7 to 1.5 us at
// 64 rows and lost 1.4 to 2.2 us at 256 (registers let one CTA of two start beside the update).
template <int HKV, bool kAfterUpdate>
__global__ void __launch_bounds__(32 * kWarps, 2) decode_q8_split_kernel(const Params p) {
  using C = Cfg<HKV>;
  constexpr int kHeads = C::kHeads, kStep = C::kStep, kRing = C::kRing, kThreads = 32 * kWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 s_ml[kWarps][kHeads][kMaxGroup];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x, b = blockIdx.y;
  const int h0 = kHeads * (warp % (HKV / kHeads));  // this warp's first kv head
  const int par = warp / (HKV / kHeads);
  const int H_Q = HKV * p.group;

  // a page in this warp's ring: K of its heads, then V, 1 KiB each
  const uint32_t ring = smem_u32(smem) + warp * (kRing * C::kPageBytes);
  const uint32_t bars = smem_u32(smem + C::kBarOffset) + warp * kRing * 8;
  if (lane == 0) {
    for (int u = 0; u < kRing; ++u) mbar_init(bars + 8 * u, 1);
    fence_mbar_init();
  }
  __syncwarp();
  // a programmatic dependent of the preceding kernel: nothing that it writes is read before
  auto wait = [] {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  };
  if (!kAfterUpdate) wait();

  // what is read before the wait comes from L2: this SM's L1 may hold older lines
  auto load = [](const auto* x) { return kAfterUpdate ? __ldcg(x) : *x; };
  const int64_t slot = load(p.slot_ids + b);
  int64_t L = kAfterUpdate ? 0 : load(p.lens + b);  // (beside the slot)
  if (slot < 0 || slot >= p.n_slots) {
    if (threadIdx.x == 0) raise_error(CIE_DEVERR_BAD_SLOT);
    L = 0;
  } else if (kAfterUpdate) {
    L = load(p.lens + slot) + 1;
  }
  if (L < 0) L = 0;
  if (L > p.row_pages * kPage) {
    if (threadIdx.x == 0) raise_error(CIE_DEVERR_BAD_LENGTH);
    L = p.row_pages * kPage;
  }
  const int Li = static_cast<int>(L), n_seq_pages = (Li + kPage - 1) / kPage;
  const int pps = decode::split_pages(n_seq_pages, p.num_splits);
  const int page_begin = split * pps;
  const int n = max(0, min(page_begin + pps, n_seq_pages) - page_begin);
  if (n == 0 && split > 0) return;  // (split 0 writes a zero row)
  const int mine = n > par ? (n - par + kStep - 1) / kStep : 0;  // pages of this warp

  // Page ids and scales of 32 of this warp's pages at a time, one per lane (the block-table
  // entries of the next 32 on their way). Scales: ks times head_dim ** -0.5 * log2(e).
  const int64_t bt_row = slot * p.bt_stride + page_begin + par;
  auto entry = [&](int i) -> int64_t {
    const int64_t at = bt_row + static_cast<int64_t>(i) * kStep;
    if (i >= mine) return 0;
    return p.table.wide ? load(static_cast<const int64_t*>(p.table.ptr) + at)
                        : load(static_cast<const int32_t*>(p.table.ptr) + at);
  };
  int64_t entry_n = entry(lane);
  int pid = 0;
  float ks[kHeads], vs[kHeads], ks_n[kHeads], vs_n[kHeads];
  const int8_t* k_base = p.k + h0 * p.head_stride;
  const int8_t* v_base = p.v + h0 * p.head_stride;
  int put = 0;  // ring place of the next page to fetch
  auto fetch = [&](int i) {
    if (i >= mine) return;
    if ((i & 31) == 0) {
      if (entry_n < 0 || entry_n >= p.n_pages) {
        raise_error(CIE_DEVERR_BAD_PAGE);
        entry_n = 0;
      }
      pid = static_cast<int>(entry_n);
    }
    const int64_t at = __shfl_sync(0xffffffffu, pid, i & 31) * p.page_stride;
    if (lane == 0) {
      const uint32_t to = ring + put * C::kPageBytes, bar = bars + 8 * put;
      mbar_arrive_expect_tx(bar, C::kPageBytes);
      if (p.head_stride == kPage * kD) {  // the heads of a page lie side by side
        copy_bulk(to, k_base + at, C::kPageBytes / 2, bar);
        copy_bulk(to + C::kPageBytes / 2, v_base + at, C::kPageBytes / 2, bar);
      } else {
        for (int u = 0; u < kHeads; ++u) {
          copy_bulk(to + 1024 * u, k_base + at + u * p.head_stride, 1024, bar);
          copy_bulk(to + 1024 * (kHeads + u), v_base + at + u * p.head_stride, 1024, bar);
        }
      }
    }
    put = put + 1 == kRing ? 0 : put + 1;
    if ((i & 31) == 0) {
      const float* sp = p.scales + static_cast<int64_t>(pid) * (2 * HKV) + h0;
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        ks_n[u] = load(sp + u) * (0.125f * kLog2e);
        vs_n[u] = load(sp + HKV + u);
      }
      entry_n = entry(i + 32 + lane);
    }
  };
  int ahead = 0;  // pages fetched before the update is done
  if (kAfterUpdate) {
    // among this warp's pages the row's last one is number `last`, if it is there at all
    const int behind = n_seq_pages - 1 - (page_begin + par);
    const int last = behind % kStep == 0 ? behind / kStep : mine;
#pragma unroll 1
    for (; ahead < min(kRing, last); ++ahead) fetch(ahead);
    wait();
    if (ahead > 0 && lane == last && last < mine) {  // its scale was read with the first 32
      const float* sp = p.scales + static_cast<int64_t>(pid) * (2 * HKV) + h0;
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        ks_n[u] = __ldcg(sp + u) * (0.125f * kLog2e);
        vs_n[u] = __ldcg(sp + HKV + u);
      }
    }
  }
#pragma unroll 1
  for (int u = ahead; u < kRing; ++u) fetch(u);

  uint32_t bq[kHeads][4][2];
  float m[kHeads][2], l[kHeads][2];  // query heads 2 t, 2 t + 1 of each kv head; m in log2
  float acc[kHeads][4][4];

  {
    // Q^T as the B operand: lane (g, t) holds query head g, dims 16 t .. 16 t + 15
    const bool valid = g < p.group;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const uint4* qr = reinterpret_cast<const uint4*>(
          p.q + (static_cast<int64_t>(b) * H_Q + (h0 + u) * p.group + (valid ? g : 0)) * kD +
          16 * t4);
      const uint4 a = valid ? qr[0] : make_uint4(0, 0, 0, 0);
      const uint4 d = valid ? qr[1] : make_uint4(0, 0, 0, 0);
      bq[u][0][0] = a.x;
      bq[u][0][1] = a.y;
      bq[u][1][0] = a.z;
      bq[u][1][1] = a.w;
      bq[u][2][0] = d.x;
      bq[u][2][1] = d.y;
      bq[u][3][0] = d.z;
      bq[u][3][1] = d.w;
      m[u][0] = m[u][1] = -CUDART_INF_F;
      l[u][0] = l[u][1] = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][e >> 2][e & 3] = 0.f;
    }
  }
  uint32_t high;
  asm volatile("mov.u32 %0, %%laneid;" : "=r"(high));
  high = (high >> 5) + 0x64646464u;  // laneid < 32
  // rows pi(g), pi(2 t) and pi(2 t + 1), and this lane's bytes of them
  const int row_g = g & 1 ? 4 + ((g >> 1) ^ 1) : g >> 1;
  const uint32_t k_at = ring + row_g * kD + 16 * t4;
  const uint32_t v_at = ring + kHeads * 1024 + t4 * kD + 8 * g;
  const uint32_t v_odd = (4 + (t4 ^ 1) - t4) * kD;  // from row pi(2 t) to row pi(2 t + 1)
  int get = 0;  // ring place of page i
  uint32_t phase = 0;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * get, phase, CIE_DEVERR_WAIT_TIMEOUT))) {
      // gave up: leave no copy in flight (each wait is bounded)
      for (int j = i; j < min(i + kRing, mine); ++j) {
        mbar_wait(bars + 8 * get, phase, CIE_DEVERR_WAIT_TIMEOUT);
        get = get + 1 == kRing ? 0 : get + 1;
        if (get == 0) phase ^= 1;
      }
      break;
    }
    if ((i & 31) == 0) {  // (fetch is less than 32 pages ahead)
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        ks[u] = ks_n[u];
        vs[u] = vs_n[u];
      }
    }
    const uint32_t page = get * C::kPageBytes;

    // scores (times log2 e): keys pi(g), pi(g) + 8 of query heads 2 t, 2 t + 1
    float s[kHeads][4];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const uint4 k0 = lds16(k_at + page + 1024 * u), k1 = lds16(k_at + page + 1024 * u + 512);
      const uint32_t* kw0 = reinterpret_cast<const uint32_t*>(&k0);
      const uint32_t* kw1 = reinterpret_cast<const uint32_t*>(&k1);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint32_t w0 = kw0[ks] ^ 0x80808080u, w1 = kw1[ks] ^ 0x80808080u;
        const uint32_t a0 = codes_to_half2(w0, 0x4140, high), a1 = codes_to_half2(w1, 0x4140, high);
        const uint32_t a2 = codes_to_half2(w0, 0x4342, high), a3 = codes_to_half2(w1, 0x4342, high);
        if (ks == 0) mma_16816_zero(s[u], a0, a1, a2, a3, bq[u][0][0], bq[u][0][1]);
        else mma_16816(s[u], a0, a1, a2, a3, bq[u][ks][0], bq[u][ks][1]);
      }
    }
    float kf[kHeads], vf[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      kf[u] = __shfl_sync(0xffffffffu, ks[u], i & 31);
      vf[u] = __shfl_sync(0xffffffffu, vs[u], i & 31);
    }
    const int rows = Li - (page_begin + par + i * kStep) * kPage;  // visible, if below 16
    float al[kHeads][2];
    bool grew = false;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][e] *= kf[u];
      if (rows < kPage) {  // rows behind the sequence's end
        if (row_g >= rows) s[u][0] = s[u][1] = -CUDART_INF_F;
        if (row_g + 8 >= rows) s[u][2] = s[u][3] = -CUDART_INF_F;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // row 0 of a page is always visible, so the new maximum is finite
        const float mn = fmaxf(m[u][e], decode::shfl_max_group(fmaxf(s[u][e], s[u][2 + e])));
        grew |= mn != m[u][e];
        al[u][e] = m[u][e] - mn;
        m[u][e] = mn;
      }
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const float a0 = ex2(al[u][0]), a1 = ex2(al[u][1]);
        l[u][0] *= a0;
        l[u][1] *= a1;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          acc[u][t][0] *= a0;
          acc[u][t][1] *= a1;
          acc[u][t][2] *= a0;
          acc[u][t][3] *= a1;
        }
      }
    }
    uint32_t pb[kHeads][2];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const float p0 = ex2(s[u][0] - m[u][0]), p1 = ex2(s[u][1] - m[u][1]);
      const float p2 = ex2(s[u][2] - m[u][0]), p3 = ex2(s[u][3] - m[u][1]);
      l[u][0] += p0 + p2;
      l[u][1] += p1 + p3;
      pb[u][0] = movmatrix_trans(pack_half2(p0, p1));
      pb[u][1] = movmatrix_trans(pack_half2(p2, p3));
    }
    // acc += scale_v * V^T . P^T
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const uint32_t va = v_at + page + 1024 * u;
      const uint2 v0 = lds8(va), v1 = lds8(va + v_odd), v2 = lds8(va + 512), v3 = lds8(va + 512 + v_odd);
#pragma unroll
      for (int wd = 0; wd < 2; ++wd) {  // dims 8 g + 4 wd .. + 3: MMA tiles 2 wd, 2 wd + 1
        const uint32_t ra = (wd ? v0.y : v0.x) ^ 0x80808080u;
        const uint32_t rb = (wd ? v1.y : v1.x) ^ 0x80808080u;
        const uint32_t rc = (wd ? v2.y : v2.x) ^ 0x80808080u;
        const uint32_t rd = (wd ? v3.y : v3.x) ^ 0x80808080u;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // dims 2 hf, 2 hf + 1 of the word
          const uint32_t sel = hf ? 0x7362 : 0x5140;  // bytes of one dim side by side
          const uint32_t ab = __byte_perm(ra, rb, sel), cd = __byte_perm(rc, rd, sel);
          float o[4];
          mma_16816_zero(o, codes_to_half2(ab, 0x4140, high), codes_to_half2(ab, 0x4342, high),
                         codes_to_half2(cd, 0x4140, high), codes_to_half2(cd, 0x4342, high), pb[u][0], pb[u][1]);
          float* d = acc[u][2 * wd + hf];
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] = fmaf(o[e], vf[u], d[e]);
        }
      }
    }
    __syncwarp();  // the page has been read
    fetch(i + kRing);
    get = get + 1 == kRing ? 0 : get + 1;
    if (get == 0) phase ^= 1;
  }

  // ---- the warps' results, merged ---------------------------------------------------
  __syncwarp();
  auto acc_of = [&](int w, int u, int hh) {  // accumulator rows in the rings
    return reinterpret_cast<float*>(smem + w * (kRing * C::kPageBytes)) +
           (u * kMaxGroup + hh) * kAccStride;
  };
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // query head 2 t + e, dims 8 g .. 8 g + 7
      const float sum = decode::shfl_sum_group(l[u][e]);
      float4* d = reinterpret_cast<float4*>(acc_of(warp, u, 2 * t4 + e) + 8 * g);
      d[0] = make_float4(acc[u][0][e], acc[u][0][2 + e], acc[u][1][e], acc[u][1][2 + e]);
      d[1] = make_float4(acc[u][2][e], acc[u][2][2 + e], acc[u][3][e], acc[u][3][2 + e]);
      if (g == 0) s_ml[warp][u][2 * t4 + e] = make_float2(m[u][e], sum);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < H_Q * (kD / 4); i += kThreads) {
    const int hq = i / (kD / 4), d4 = i % (kD / 4);
    const int kv = hq / p.group, hh = hq - kv * p.group, u = kv % kHeads, w0 = kv / kHeads;
    float2 ml[kStep];
    float M = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kStep; ++w) {
      ml[w] = s_ml[w * (HKV / kHeads) + w0][u][hh];
      M = fmaxf(M, ml[w].x);
    }
    float sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n > 0) {
#pragma unroll
      for (int w = 0; w < kStep; ++w) {
        const float wt = ex2(ml[w].x - M);  // 0 of a warp that saw no page
        const float4 x = *reinterpret_cast<const float4*>(
            acc_of(w * (HKV / kHeads) + w0, u, hh) + 4 * d4);
        sum += wt * ml[w].y;
        a.x += wt * x.x;
        a.y += wt * x.y;
        a.z += wt * x.z;
        a.w += wt * x.w;
      }
    }
    if (n == n_seq_pages) {
      const float inv = n > 0 ? 1.f / sum : 0.f;  // a row that saw no key is zero
      uint2 r;
      r.x = pack_half2(a.x * inv, a.y * inv);
      r.y = pack_half2(a.z * inv, a.w * inv);
      *reinterpret_cast<uint2*>(p.o + (static_cast<int64_t>(b) * H_Q + hq) * kD + 4 * d4) = r;
    } else {
      const int64_t row = (static_cast<int64_t>(b) * p.num_splits + split) * H_Q + hq;
      *reinterpret_cast<float4*>(p.ws_acc + row * kD + 4 * d4) = a;
      if (d4 == 0) *reinterpret_cast<float2*>(p.ws_ml + row * 2) = make_float2(M, sum);
    }
  }
}

// Merges the partials of the sequences that have several splits: O = sum_s w_s acc_s /
// sum_s w_s l_s, w_s = 2^(m_s - max m). kFold > 1: a CTA of kFold warps per (query head,
// sequence), each folding every kFold-th split; 1: a CTA per sequence, a warp per query
// head. A lane holds two columns. A programmatic dependent of the split kernel.
template <int HKV, int kFold>
__global__ void __launch_bounds__(kFold > 1 ? 32 * kFold : 1024) merge_q8_kernel(const Params p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H_Q = HKV * p.group;
  const int b = blockIdx.x, hq = kFold > 1 ? blockIdx.y : warp, fold = kFold > 1 ? warp : 0;
  // (the split kernel does not write slots and lengths; read past L1)
  const int n = seq_pages(p, b);
  const int pps = decode::split_pages(n, p.num_splits);
  // Every CTA waits, also one with nothing to merge: a grid that ended without waiting
  // would let the kernel after it start while the split kernel still writes its rows.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n <= pps) return;
  const int splits = (n + pps - 1) / pps;
  float M = -CUDART_INF_F, l = 0.f;
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int s = fold; s < splits; s += kFold) {
    const int64_t row = (static_cast<int64_t>(b) * p.num_splits + s) * H_Q + hq;
    const float2 ml = *reinterpret_cast<const float2*>(p.ws_ml + row * 2);
    const float2 a = *reinterpret_cast<const float2*>(p.ws_acc + row * kD + 2 * lane);
    const float Mn = fmaxf(M, ml.x);  // finite: every split saw a key
    const float wo = ex2(M - Mn), wn = ex2(ml.x - Mn);
    l = l * wo + ml.y * wn;
    acc.x = acc.x * wo + a.x * wn;
    acc.y = acc.y * wo + a.y * wn;
    M = Mn;
  }
  if (kFold > 1) {
    __shared__ float s_m[kFold], s_l[kFold];
    __shared__ float2 s_acc[kFold][32];
    if (lane == 0) {
      s_m[fold] = M;
      s_l[fold] = l;
    }
    s_acc[fold][lane] = acc;
    __syncthreads();
    if (fold != 0) return;
    for (int w = 1; w < min(kFold, splits); ++w) {
      const float Mn = fmaxf(M, s_m[w]);
      const float wo = ex2(M - Mn), wn = ex2(s_m[w] - Mn);
      l = l * wo + s_l[w] * wn;
      acc.x = acc.x * wo + s_acc[w][lane].x * wn;
      acc.y = acc.y * wo + s_acc[w][lane].y * wn;
      M = Mn;
    }
  }
  const float inv = 1.f / l;
  *reinterpret_cast<__half2*>(p.o + (static_cast<int64_t>(b) * H_Q + hq) * kD + 2 * lane) =
      __floats2half2_rn(acc.x * inv, acc.y * inv);
}

template <int HKV, bool kAfterUpdate>
int launch(const Params& p, int batch, cudaStream_t stream) {
  const auto split_kernel = decode_q8_split_kernel<HKV, kAfterUpdate>;
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(split_kernel),
                                       Cfg<HKV>::kSmemBytes, (kAfterUpdate ? 14 : 10) + HKV);
  if (st != CIE_OK) return st;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.num_splits, batch);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = Cfg<HKV>::kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, split_kernel, p);
  if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "decode_q8 launch: %s", cudaGetErrorString(e));
  if (p.num_splits > 1) {
    const int H_Q = HKV * p.group;
    const bool wide = p.num_splits > 16;  // few sequences, many splits
    cfg.gridDim = wide ? dim3(batch, H_Q) : dim3(batch);
    cfg.blockDim = dim3(wide ? 256 : 32 * H_Q);
    cfg.dynamicSmemBytes = 0;
    e = wide ? cudaLaunchKernelEx(&cfg, merge_q8_kernel<HKV, 8>, p)
             : cudaLaunchKernelEx(&cfg, merge_q8_kernel<HKV, 1>, p);
    if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "merge launch: %s", cudaGetErrorString(e));
  }
  return CIE_OK;
}

// Checks of a call; sets what is common to both entry points. `q_bytes` of the workspace
// lie in front of the partials.
int prepare(Params& p, const void* q, const void* k, const void* v, const float* kv_scales,
            const int64_t* lens, const int64_t* slot_ids, BlockTable table, void* o,
            void* workspace, size_t workspace_bytes, size_t q_bytes, int batch, int num_q_heads,
            int num_kv_heads, int head_dim, int page_size, int64_t n_pages, int64_t n_slots,
            int64_t bt_stride, int64_t page_stride, int64_t head_stride, int num_splits) {
  if (!q || !lens || !slot_ids || !table.ptr || !o)
    return fail(CIE_ERR_INVALID_ARGUMENT, "null pointer argument");
  const int st = kvq8::check_pool(k, v, kv_scales, num_kv_heads, head_dim, page_size, n_pages,
                                  n_slots, bt_stride, page_stride, head_stride);
  if (st != CIE_OK) return st;
  if (num_kv_heads != 1 && num_kv_heads != 2 && num_kv_heads != 4)
    return fail(CIE_ERR_UNSUPPORTED, "num_kv_heads %d (supported: 1, 2, 4)", num_kv_heads);
  if (num_q_heads < num_kv_heads || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > kMaxGroup)
    return fail(CIE_ERR_UNSUPPORTED, "num_q_heads %d must be 1 to 8 times num_kv_heads",
                num_q_heads);
  if (n_pages >= (int64_t(1) << 31) || bt_stride >= (int64_t(1) << 27))
    return fail(CIE_ERR_OVERFLOW, "n_pages %lld / bt_stride %lld do not fit int32",
                (long long)n_pages, (long long)bt_stride);
  if (batch > 65535) return fail(CIE_ERR_UNSUPPORTED, "batch %d > 65535", batch);
  if (!aligned16(q) || !aligned16(o)) return fail(CIE_ERR_ALIGNMENT, "q / o must be 16-byte aligned");
  const int S = num_splits > 0 ? num_splits : cie_decode_q8_default_splits(batch, current_device());
  if (S > 4096) return fail(CIE_ERR_INVALID_ARGUMENT, "num_splits %d > 4096", S);
  const size_t need =
      q_bytes + (S > 1 ? cie_decode_workspace_bytes(batch, num_q_heads, head_dim, S) : 0);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail(CIE_ERR_WORKSPACE, "the call needs %zu workspace bytes, got %zu", need,
                  workspace == nullptr ? size_t(0) : workspace_bytes);
    if (!aligned16(workspace)) return fail(CIE_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    p.ws_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + q_bytes);
    p.ws_ml = p.ws_acc + static_cast<int64_t>(batch) * S * num_q_heads * kD;
  }
  p.q = static_cast<const __half*>(q);
  p.k = static_cast<const int8_t*>(k);
  p.v = static_cast<const int8_t*>(v);
  p.scales = kv_scales;
  p.lens = lens;
  p.slot_ids = slot_ids;
  p.table = table;
  p.o = static_cast<__half*>(o);
  p.num_splits = S;
  p.group = num_q_heads / num_kv_heads;
  p.n_pages = n_pages;
  p.n_slots = n_slots;
  p.bt_stride = bt_stride;
  p.row_pages = kvq8::row_pages(bt_stride, n_pages);
  p.page_stride = page_stride;
  p.head_stride = head_stride;
  return CIE_OK;
}

template <bool kAfterUpdate>
int run(const Params& p, int batch, int num_kv_heads, cie_stream_t stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (num_kv_heads) {
    case 1: return launch<1, kAfterUpdate>(p, batch, s);
    case 2: return launch<2, kAfterUpdate>(p, batch, s);
    default: return launch<4, kAfterUpdate>(p, batch, s);
  }
}

int entry(const void* q, const void* k, const void* v, const float* kv_scales,
          const int64_t* lens, const int64_t* slot_ids, BlockTable table, void* o,
          void* workspace, size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads,
          int head_dim, int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
          int64_t page_stride, int64_t head_stride, int num_splits, cie_stream_t stream) {
  if (batch < 0) return fail(CIE_ERR_INVALID_ARGUMENT, "batch < 0");
  if (batch == 0) return CIE_OK;
  Params p{};
  const int st = prepare(p, q, k, v, kv_scales, lens, slot_ids, table, o, workspace,
                         workspace_bytes, 0, batch, num_q_heads, num_kv_heads, head_dim,
                         page_size, n_pages, n_slots, bt_stride, page_stride, head_stride,
                         num_splits);
  return st != CIE_OK ? st : run<false>(p, batch, num_kv_heads, stream);
}

// Rotated q in front of the split scratch.
size_t q_bytes(int batch, int num_q_heads, int head_dim) {
  return static_cast<size_t>(batch) * num_q_heads * head_dim * sizeof(__half);
}

int rope_entry(const void* qkv, int64_t qkv_tok, const void* cos, const void* sin,
               int64_t cs_tok, void* k, void* v, float* kv_scales, const int64_t* lens,
               const int64_t* slot_ids, BlockTable table, void* o, void* workspace,
               size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads,
               int head_dim, int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
               int64_t page_stride, int64_t head_stride, int num_splits, cie_stream_t stream) {
  if (batch < 0) return fail(CIE_ERR_INVALID_ARGUMENT, "batch < 0");
  if (batch == 0) return CIE_OK;
  if (!workspace) return fail(CIE_ERR_WORKSPACE, "no workspace");
  Params p{};
  int st = prepare(p, workspace, k, v, kv_scales, lens, slot_ids, table, o, workspace,
                   workspace_bytes, q_bytes(batch, num_q_heads, kD), batch, num_q_heads,
                   num_kv_heads, head_dim, page_size, n_pages, n_slots, bt_stride, page_stride,
                   head_stride, num_splits);
  if (st != CIE_OK) return st;
  p.after_update = 1;
  kvq8::Args a = kvq8::pool_args(k, v, kv_scales, slot_ids, table, batch, num_kv_heads, n_pages,
                                 n_slots, bt_stride, page_stride, head_stride);
  kvq8::set_rope(a, qkv, qkv_tok, cos, sin, cs_tok, workspace, num_q_heads);
  a.lens = lens;
  a.tokens = batch;
  st = kvq8::update(a, true, false, head_dim, page_size, stream);
  return st != CIE_OK ? st : run<true>(p, batch, num_kv_heads, stream);
}

}  // namespace dq8
}  // namespace cie

extern "C" {

int cie_decode_q8_default_splits(int batch, int device) {
  int sms = 148;
  if (device >= 0 && device == cie::current_device()) {
    sms = cie::sm_count();  // (remembered)
  } else if (device >= 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess && n > 0)
      sms = n;
  }
  if (batch <= 0) return 1;
  // Two CTAs per SM, as the smallest power of two that is at least 4/5 of that, and 64 at
  // most. More CTAs even out ragged batches, where the longest split sets the time (256
  // sequences of 1 to 4096 rows, one kv head: 32 us at 1 split, 29 at 2, 31 at 4; 100 of 1 to
  // 4000, four heads: 50 at 2, 38 at 4), but cost even ones a second wave and a merge
  // (256 x 4096, two heads: 53 us at 1 split, 58 at 2; 64 x 4096: 20 at 4, 24 at 8). The cap
  // leaves one or two sequences 64 or 128 CTAs of the 296 places: right up to 16384 rows (one:
  // 7.4 us at 64, 7.9 at 128; two: 7.6 and 9.2) and about even at 32768 (9.2 and 8.7; 10.2 and
  // 11.4); one of 131072 rows would take 15.6 us at 128 instead of 21.7, two 20.9 instead of 22.2.
  int s = 1;
  while (s < 64 && 5LL * s * batch < 8LL * sms) s *= 2;
  return s;
}

int cie_decode_attention_q8(const void* q, const void* k, const void* v, const float* kv_scales,
                            const int64_t* lens, const int64_t* slot_ids,
                            const int64_t* block_table, void* o, void* workspace,
                            size_t workspace_bytes, int batch, int num_q_heads,
                            int num_kv_heads, int head_dim, int page_size, int64_t n_pages,
                            int64_t n_slots, int64_t bt_stride, int64_t kv_page_stride,
                            int64_t kv_head_stride, int num_splits, cie_stream_t stream) {
  return cie::dq8::entry(q, k, v, kv_scales, lens, slot_ids, cie::BlockTable{block_table, 1}, o,
                         workspace, workspace_bytes, batch, num_q_heads, num_kv_heads, head_dim,
                         page_size, n_pages, n_slots, bt_stride, kv_page_stride, kv_head_stride,
                         num_splits, stream);
}

int cie_decode_attention_q8_bt32(const void* q, const void* k, const void* v,
                                 const float* kv_scales, const int64_t* lens,
                                 const int64_t* slot_ids, const int32_t* block_table, void* o,
                                 void* workspace, size_t workspace_bytes, int batch,
                                 int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                 int64_t n_pages, int64_t n_slots, int64_t bt_stride,
                                 int64_t kv_page_stride, int64_t kv_head_stride, int num_splits,
                                 cie_stream_t stream) {
  return cie::dq8::entry(q, k, v, kv_scales, lens, slot_ids, cie::BlockTable{block_table, 0}, o,
                         workspace, workspace_bytes, batch, num_q_heads, num_kv_heads, head_dim,
                         page_size, n_pages, n_slots, bt_stride, kv_page_stride, kv_head_stride,
                         num_splits, stream);
}

size_t cie_rope_kv_q8_decode_workspace_bytes(int batch, int num_q_heads, int head_dim,
                                             int num_splits) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0) return 0;
  return cie::dq8::q_bytes(batch, num_q_heads, head_dim) +
         (num_splits > 1 ? cie_decode_workspace_bytes(batch, num_q_heads, head_dim, num_splits) : 0);
}

int cie_rope_kv_q8_decode_attention(
    const void* qkv, int64_t qkv_tok_stride, const void* cos, const void* sin,
    int64_t cs_tok_stride, void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
    const int64_t* slot_ids, const int64_t* block_table, void* o, void* workspace,
    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim,
    int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, int num_splits, cie_stream_t stream) {
  return cie::dq8::rope_entry(qkv, qkv_tok_stride, cos, sin, cs_tok_stride, k_cache, v_cache,
                              kv_scales, lens, slot_ids, cie::BlockTable{block_table, 1}, o,
                              workspace, workspace_bytes, batch, num_q_heads, num_kv_heads,
                              head_dim, page_size, n_pages, n_slots, bt_stride,
                              cache_page_stride, cache_head_stride, num_splits, stream);
}

int cie_rope_kv_q8_decode_attention_bt32(
    const void* qkv, int64_t qkv_tok_stride, const void* cos, const void* sin,
    int64_t cs_tok_stride, void* k_cache, void* v_cache, float* kv_scales, const int64_t* lens,
    const int64_t* slot_ids, const int32_t* block_table, void* o, void* workspace,
    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim,
    int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
    int64_t cache_page_stride, int64_t cache_head_stride, int num_splits, cie_stream_t stream) {
  return cie::dq8::rope_entry(qkv, qkv_tok_stride, cos, sin, cs_tok_stride, k_cache, v_cache,
                              kv_scales, lens, slot_ids, cie::BlockTable{block_table, 0}, o,
                              workspace, workspace_bytes, batch, num_q_heads, num_kv_heads,
                              head_dim, page_size, n_pages, n_slots, bt_stride,
                              cache_page_stride, cache_head_stride, num_splits, stream);
}

}  // extern "C"
