// Split-KV paged GQA decode attention over 8-bit pages (sm_100a).
//
// One CTA per (split, sequence), eight warps; a warp takes one kv head of every
// (8 / HKV)-th page of the split, so its working set is one K tile and one V
// tile of 16 rows x 64 codes (1 KiB each). The tiles go from global memory
// straight to registers, kPrefetch pages ahead. Nothing is staged in shared
// memory, and no thread issues copies for others: half the bytes a page means
// twice the pages a second, and one thread issuing bulk copies of 2 KiB would
// bound the CTA (a single issuer of 4 KiB copies streams about 30 GB/s).
//
// Mathematics, per page and kv head (16 keys, up to 8 query heads on the MMA's N
// side), warp-level MMA with fp16 operands and fp32 accumulation:
//   S^T (16 x 8) = Kc (16 x 64) . Q^T (64 x 8),  s = S^T * scale_k / 8
//   online softmax over keys in fp32; p = exp(s - m), rounded to fp16
//   O^T (64 x 8) = alpha O^T + scale_v * (Vc^T (64 x 16) . P^T (16 x 8))
// Codes are whole numbers up to 127, exact in fp16: a byte c + 128 under the
// exponent byte 0x64 is the fp16 number 1024 + 128 + c, and subtracting 1152 is
// exact. scale_k and scale_v multiply fp32 results, so neither p nor a code is
// ever scaled in fp16, whatever range the page scales span.
//
// Contraction indices and output rows may be numbered freely as long as both
// operands agree, so every lane's operand bytes are contiguous in memory:
//   S: lane (g, t) loads bytes [16 t, 16 t + 16) of rows pi(g) and pi(g) + 8;
//      MMA step ks contracts dims 16 t + 4 ks + {0, 1, 2, 3}
//   O: lane (g, t) loads bytes [8 g, 8 g + 8) of rows t, 4 + t, 8 + t, 12 + t, which
//      are MMA keys 2t, 2t + 1, 2t + 8, 2t + 9; MMA row g of tile mt is dim 8 g + 2 mt,
//      row g + 8 is dim 8 g + 2 mt + 1
// with pi(2 t) = t, pi(2 t + 1) = 4 + t.
#include "cie_common.cuh"
#include "cie_host.h"
#include "cie_kv_q8.h"

namespace cie {
namespace dq8 {

constexpr int kD = 64;
constexpr int kPage = 16;
constexpr int kWarps = 8;
constexpr int kMaxGroup = 8;
constexpr int kPrefetch = 2;
constexpr int kAccStride = kD + 4;  // floats of one head in the merge buffer (banks)

struct Params {
  const __half* q;          // (B, H_q, D)
  const int8_t* k;          // (n_pages, HKV, 16, 64)
  const int8_t* v;
  const float* scales;      // (n_pages, 2, HKV)
  const int64_t* lens;      // (B,)
  const int64_t* slot_ids;  // (B,)
  BlockTable table;         // (n_slots, bt_stride)
  __half* o;                // (B, H_q, D)
  float* ws_acc;            // (B, S, H_q, D)
  float* ws_ml;             // (B, S, H_q, 2)
  int num_splits;
  int group;                // query heads per kv head, 1..8
  int64_t n_pages, n_slots, bt_stride;
  int64_t page_stride, head_stride;
};

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__device__ __forceinline__ uint2 ld_stream8(const void* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// Two biased codes of `w` (code + 128, picked by the selector) as a pair of fp16.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w, uint32_t sel) {
  uint32_t h = __byte_perm(w, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&h), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// One page of one kv head, as loaded.
struct Tile {
  uint4 k0, k1;             // rows pi(g), pi(g) + 8
  uint2 v[4];               // rows t, 4 + t, 8 + t, 12 + t
  float ks, vs;             // scales
};

template <int HKV>
__global__ void __launch_bounds__(32 * kWarps, 2) decode_q8_split_kernel(const Params p) {
  constexpr int kStep = kWarps / HKV;  // warps per kv head: pages apart
  __shared__ float s_acc[kWarps][kMaxGroup][kAccStride];
  __shared__ float s_m[kWarps][kMaxGroup], s_l[kWarps][kMaxGroup];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x, b = blockIdx.y, S = p.num_splits;
  const int h = warp % HKV, par = warp / HKV;
  const int H_Q = HKV * p.group;

  // a programmatic dependent of the preceding kernel: no input is read before this
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int64_t slot = p.slot_ids[b];
  int64_t L = p.lens[b];
  if (slot < 0 || slot >= p.n_slots) {
    if (threadIdx.x == 0) raise_error(CIE_DEVERR_BAD_SLOT);
    L = 0;
  }
  if (L < 0) L = 0;
  if ((L + kPage - 1) / kPage > p.bt_stride) {
    if (threadIdx.x == 0) raise_error(CIE_DEVERR_BAD_LENGTH);
    L = p.bt_stride * kPage;
  }
  const int n_seq_pages = static_cast<int>((L + kPage - 1) / kPage);
  const int pps = decode::split_pages(n_seq_pages, S);
  const int page_begin = split * pps;
  const int n = max(0, min(page_begin + pps, n_seq_pages) - page_begin);
  const int Li = static_cast<int>(L);
  const int mine = n > par ? (n - par + kStep - 1) / kStep : 0;  // pages of this warp

  // Page ids and scales of 32 of this warp's pages at a time, one per lane: the
  // batch in use, the ids of the next one (whose scales are on their way) and the
  // table entries of the one after.
  const int64_t bt_row = slot * p.bt_stride + page_begin;
  auto entry = [&](int i) -> int64_t {
    return i < mine ? p.table.at(bt_row + par + static_cast<int64_t>(i) * kStep) : 0;
  };
  auto checked = [&](int64_t pid) -> int {
    if (pid < 0 || pid >= p.n_pages) {
      raise_error(CIE_DEVERR_BAD_PAGE);
      return 0;
    }
    return static_cast<int>(pid);
  };
  int pid_c = 0, pid_n = 0;
  float ks_c = 0.f, vs_c = 0.f, ks_n = 0.f, vs_n = 0.f;
  int64_t e_nn = 0;
  auto load_scales = [&](int pid, float& ks, float& vs) {
    const float* sp = p.scales + static_cast<int64_t>(pid) * (2 * HKV) + h;
    ks = sp[0];
    vs = sp[HKV];
  };

  Tile tile[kPrefetch];
  auto fetch = [&](Tile& x, int i) {  // page i of this warp; i counts up from 0
    if (i >= mine) return;
    if (i != 0 && (i & 31) == 0) {
      pid_c = pid_n;
      ks_c = ks_n;
      vs_c = vs_n;
      pid_n = checked(e_nn);
      load_scales(pid_n, ks_n, vs_n);
      e_nn = entry(i + 64 + lane);
    }
    const int pid = __shfl_sync(0xffffffffu, pid_c, i & 31);
    x.ks = __shfl_sync(0xffffffffu, ks_c, i & 31);
    x.vs = __shfl_sync(0xffffffffu, vs_c, i & 31);
    const int64_t at = static_cast<int64_t>(pid) * p.page_stride + h * p.head_stride;
    const int8_t* kp = p.k + at + ((g >> 1) + 4 * (g & 1)) * kD + 16 * t4;
    x.k0 = ld_stream16(kp);
    x.k1 = ld_stream16(kp + 8 * kD);
    const int8_t* vp = p.v + at + t4 * kD + 8 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = ld_stream8(vp + 4 * j * kD);
  };
  if (mine > 0) {
    pid_c = checked(entry(lane));
    load_scales(pid_c, ks_c, vs_c);
    pid_n = checked(entry(32 + lane));
    load_scales(pid_n, ks_n, vs_n);
    e_nn = entry(64 + lane);
#pragma unroll
    for (int u = 0; u < kPrefetch; ++u) fetch(tile[u], u);
  }

  // Q^T as the B operand: lane (g, t) holds query head g, dims 16 t .. 16 t + 15
  uint32_t bq[4][2];
  {
    const bool valid = g < p.group;
    const uint4* qr = reinterpret_cast<const uint4*>(
        p.q + (static_cast<int64_t>(b) * H_Q + h * p.group + (valid ? g : 0)) * kD + 16 * t4);
    const uint4 a = valid ? qr[0] : make_uint4(0, 0, 0, 0);
    const uint4 c = valid ? qr[1] : make_uint4(0, 0, 0, 0);
    bq[0][0] = a.x;
    bq[0][1] = a.y;
    bq[1][0] = a.z;
    bq[1][1] = a.w;
    bq[2][0] = c.x;
    bq[2][1] = c.y;
    bq[3][0] = c.z;
    bq[3][1] = c.w;
  }

  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F;  // heads 2 t, 2 t + 1
  float l0 = 0.f, l1 = 0.f;
  float acc[4][4];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[mt][e] = 0.f;

  auto step = [&](const Tile& x, int i) {
    float sc[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t* kw0 = reinterpret_cast<const uint32_t*>(&x.k0);
    const uint32_t* kw1 = reinterpret_cast<const uint32_t*>(&x.k1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const uint32_t w0 = kw0[ks] ^ 0x80808080u, w1 = kw1[ks] ^ 0x80808080u;
      mma_16816(sc, codes_to_half2(w0, 0x4140), codes_to_half2(w1, 0x4140),
                codes_to_half2(w0, 0x4342), codes_to_half2(w1, 0x4342), bq[ks][0], bq[ks][1]);
    }
    const float f = x.ks * 0.125f;  // head_dim ** -0.5 for D = 64
    float s0 = sc[0] * f, s1 = sc[1] * f, s2 = sc[2] * f, s3 = sc[3] * f;
    const int first = (page_begin + par + i * kStep) * kPage;
    if (first + kPage > Li) {  // the sequence's last page: rows beyond its end
      const int key0 = first + (g >> 1) + 4 * (g & 1);
      if (key0 >= Li) s0 = s1 = -CUDART_INF_F;
      if (key0 + 8 >= Li) s2 = s3 = -CUDART_INF_F;
    }
    const float mn0 = fmaxf(m0, decode::shfl_max_group(fmaxf(s0, s2)));
    const float mn1 = fmaxf(m1, decode::shfl_max_group(fmaxf(s1, s3)));
    if (__any_sync(0xffffffffu, mn0 != m0 || mn1 != m1)) {
      // row 0 of a visited page is always visible, so mn0 and mn1 are finite here
      const float al0 = ex2((m0 - mn0) * kLog2e);
      const float al1 = ex2((m1 - mn1) * kLog2e);
      l0 *= al0;
      l1 *= al1;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        acc[mt][0] *= al0;
        acc[mt][1] *= al1;
        acc[mt][2] *= al0;
        acc[mt][3] *= al1;
      }
      m0 = mn0;
      m1 = mn1;
    }
    const float p0 = ex2((s0 - m0) * kLog2e);
    const float p1 = ex2((s1 - m1) * kLog2e);
    const float p2 = ex2((s2 - m0) * kLog2e);
    const float p3 = ex2((s3 - m1) * kLog2e);
    l0 += p0 + p2;
    l1 += p1 + p3;
    const uint32_t pb0 = movmatrix_trans(pack_half2(p0, p1));
    const uint32_t pb1 = movmatrix_trans(pack_half2(p2, p3));
#pragma unroll
    for (int wd = 0; wd < 2; ++wd) {  // dims 8 g + 4 wd .. + 3: MMA tiles 2 wd, 2 wd + 1
      const uint32_t ra = (wd ? x.v[0].y : x.v[0].x) ^ 0x80808080u;
      const uint32_t rb = (wd ? x.v[1].y : x.v[1].x) ^ 0x80808080u;
      const uint32_t rc = (wd ? x.v[2].y : x.v[2].x) ^ 0x80808080u;
      const uint32_t rd = (wd ? x.v[3].y : x.v[3].x) ^ 0x80808080u;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {  // dims 2 hf, 2 hf + 1 of the word
        const uint32_t sel = hf ? 0x7362 : 0x5140;  // bytes of one dim side by side
        const uint32_t ab = __byte_perm(ra, rb, sel), cd = __byte_perm(rc, rd, sel);
        float o[4] = {0.f, 0.f, 0.f, 0.f};
        mma_16816(o, codes_to_half2(ab, 0x4140), codes_to_half2(ab, 0x4342),
                  codes_to_half2(cd, 0x4140), codes_to_half2(cd, 0x4342), pb0, pb1);
        float* d = acc[2 * wd + hf];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = fmaf(o[e], x.vs, d[e]);
      }
    }
  };

  for (int i = 0; i < mine; i += kPrefetch) {
#pragma unroll
    for (int u = 0; u < kPrefetch; ++u) {
      if (i + u < mine) step(tile[u], i + u);
      fetch(tile[u], i + u + kPrefetch);
    }
  }
  l0 = decode::shfl_sum_group(l0);
  l1 = decode::shfl_sum_group(l1);

  // ---- the warps of a kv head, merged -----------------------------------------
#pragma unroll
  for (int e = 0; e < 2; ++e) {  // heads 2 t + e, dims 8 g .. 8 g + 7
    float4* d = reinterpret_cast<float4*>(&s_acc[warp][2 * t4 + e][8 * g]);
    d[0] = make_float4(acc[0][e], acc[0][2 + e], acc[1][e], acc[1][2 + e]);
    d[1] = make_float4(acc[2][e], acc[2][2 + e], acc[3][e], acc[3][2 + e]);
  }
  if (g == 0) {
    s_m[warp][2 * t4] = m0;
    s_m[warp][2 * t4 + 1] = m1;
    s_l[warp][2 * t4] = l0;
    s_l[warp][2 * t4 + 1] = l1;
  }
  __syncthreads();
  if (S > 1 && n == 0) return;  // the merge reads only splits that saw pages
  for (int i = threadIdx.x; i < HKV * p.group * (kD / 4); i += 32 * kWarps) {
    const int hq = i / (kD / 4), d4 = i % (kD / 4);
    const int kv = hq / p.group, hh = hq % p.group;
    float M = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kStep; ++w) M = fmaxf(M, s_m[w * HKV + kv][hh]);
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (M != -CUDART_INF_F) {
#pragma unroll
      for (int w = 0; w < kStep; ++w) {
        const float wt = ex2((s_m[w * HKV + kv][hh] - M) * kLog2e);
        const float4 x = *reinterpret_cast<const float4*>(&s_acc[w * HKV + kv][hh][4 * d4]);
        l += wt * s_l[w * HKV + kv][hh];
        a.x += wt * x.x;
        a.y += wt * x.y;
        a.z += wt * x.z;
        a.w += wt * x.w;
      }
    }
    if (S == 1) {
      const float inv = l > 0.f ? 1.f / l : 0.f;  // a row that saw no key is zero
      uint2 r;
      r.x = pack_half2(a.x * inv, a.y * inv);
      r.y = pack_half2(a.z * inv, a.w * inv);
      *reinterpret_cast<uint2*>(p.o + (static_cast<int64_t>(b) * H_Q + hq) * kD + 4 * d4) = r;
    } else {
      const int64_t row = (static_cast<int64_t>(b) * S + split) * H_Q + hq;
      *reinterpret_cast<float4*>(p.ws_acc + row * kD + 4 * d4) = a;
      if (d4 == 0) {
        p.ws_ml[row * 2] = M;
        p.ws_ml[row * 2 + 1] = l;
      }
    }
  }
}

template <int HKV>
int launch(const Params& p, int batch, cudaStream_t stream) {
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.num_splits, batch);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, decode_q8_split_kernel<HKV>, p);
  if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "decode_q8 launch: %s", cudaGetErrorString(e));
  if (p.num_splits > 1) {
    const int H_Q = HKV * p.group;
    const bool small = p.num_splits <= decode::kSmallMergeSplits;
    cfg.gridDim = small ? dim3(batch) : dim3(H_Q, batch);
    cfg.blockDim = dim3(small ? 32 * H_Q : 256);
    e = cudaLaunchKernelEx(&cfg,
                           small ? decode::decode_merge_small_kernel : decode::decode_merge_kernel,
                           static_cast<const float*>(p.ws_acc),
                           static_cast<const float*>(p.ws_ml), p.o, p.lens, p.slot_ids,
                           p.n_slots, p.bt_stride, p.num_splits, H_Q, 0);
    if (e != cudaSuccess) return fail(CIE_ERR_CUDA, "merge launch: %s", cudaGetErrorString(e));
  }
  return CIE_OK;
}

int entry(const void* q, const void* k, const void* v, const float* kv_scales,
          const int64_t* lens, const int64_t* slot_ids, BlockTable table, void* o,
          void* workspace, size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads,
          int head_dim, int page_size, int64_t n_pages, int64_t n_slots, int64_t bt_stride,
          int64_t page_stride, int64_t head_stride, int num_splits, cie_stream_t stream) {
  if (batch < 0) return fail(CIE_ERR_INVALID_ARGUMENT, "batch < 0");
  if (batch == 0) return CIE_OK;
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
  Params p{};
  if (S > 1) {
    const size_t need = cie_decode_workspace_bytes(batch, num_q_heads, head_dim, S);
    if (workspace == nullptr || workspace_bytes < need)
      return fail(CIE_ERR_WORKSPACE, "split path needs %zu workspace bytes, got %zu", need,
                  workspace == nullptr ? size_t(0) : workspace_bytes);
    if (!aligned16(workspace)) return fail(CIE_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    p.ws_acc = static_cast<float*>(workspace);
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
  p.page_stride = page_stride;
  p.head_stride = head_stride;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (num_kv_heads) {
    case 1: return launch<1>(p, batch, s);
    case 2: return launch<2>(p, batch, s);
    default: return launch<4>(p, batch, s);
  }
}

}  // namespace dq8
}  // namespace cie

extern "C" {

int cie_decode_q8_default_splits(int batch, int device) {
  return cie_decode_default_splits(batch, device);
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

}  // extern "C"
