// Batched paged GQA decode attention over an 8-bit cache: K and V pools of e4m3 values with one
// scale per (page, KV head), one query token per request.
//
//   out[b, hq] = sum_t p_t sv(t) V[t] / sum_t p_t,   p_t = exp(scale * sk(t) q . K[t] - max)
//
// What bounds it: K and V once, HBM. At half the bytes of a 16-bit cache the arithmetic per
// byte doubles, so the values are never widened: both products run on the tensor cores in e4m3
// (mma.sync m16n8k32, which measured 0.90 per clock and SM here against 0.48 for the 16-bit
// m16n8k16), and the 16-bit operands are split into e4m3 parts whose sum they are:
//   q 2^k = q1 + q2 (+ q3),  each part the e4m3 rounding of what the ones before leave.
// A bf16 value has 8 significant bits and two parts hold it exactly (down to 2^-18 of the row's
// largest element); an f16 value has 11 and takes three. P is split the same way (two parts:
// 2^-8 relative, as near as bf16; three for f16: 2^-12). The parts ride in the n dimension: up to
// four query heads per KV head, part 1 is columns 0-3 and part 2 columns 4-7 of one MMA.
//
// A step of a warp is a unit of 32 tokens (two pages of 16, or one of 32):
//   S^T[tokens, cols] = K[tokens, D] . Q^T            A = K by ldmatrix, rows of 32 bytes
//   softmax of the unit against its own maximum, then
//   O^T[D, cols] = alpha O^T + beta (V^T[D, tokens] . P^T[tokens, cols])
//                                                     A = V^T by ldmatrix .b8 transposed
// P is relative to the unit's maximum and to its larger V scale, times 256: e4m3's range covers
// every unit alike, whatever the running maximum, and what P loses below 2^-18 of the unit's
// largest weight stays below 2^-18 of that unit's share. beta = 2^(max_unit - max) sv.
// The S^T accumulator becomes the P^T operand with one movmatrix per 16 tokens: a 16-bit element
// carries the bytes of two tokens, and the token order that leaves is made good by the row
// addresses of V's ldmatrix. The MMA rows 8..15 are tokens 12..15, 8..11, which keeps both K's
// and V's ldmatrix free of bank conflicts in the 128-byte swizzle.
//
// Work: the stream of units over (request, KV head) is cut into equal ranges, one per resident
// warp, each with its own ring of TMA stages; pieces of a cut (request, head) are merged by the
// last warp to finish one (the counters return to zero). More than eight query heads per KV
// head run as several passes over it.
//
// Generic kernel (fp32 queries, other head sizes and pages): one CTA per (request, query head).
#include <atomic>
#include <type_traits>

#include <cuda_fp8.h>
#include <cudaTypedefs.h>

#include "pi_common.cuh"

namespace pi {
namespace attn {
PFN_cuTensorMapEncodeTiled_v12000 get_encode();  // paged_decode_attn.cu
}  // namespace attn

namespace q8 {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 32;            // tokens per step
constexpr int kMaxBatch = 4096;
constexpr int kMaxSegments = 4096 * 64;  // arrival counters
constexpr int kMaxCtasPerSm = 2;
constexpr int kHeadsPad = 8;
constexpr unsigned kFull = 0xffffffffu;

struct Params {
  void* out;
  const void* q;
  const float* k_scale;  // [num_pages, hkv]
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* ctx_lens;
  int64_t bt_stride;
  int64_t q_stride;
  int64_t out_stride;
  int64_t num_pages;
  int batch, max_pages, hkv;
  int group;   // query heads per KV head
  int passes;  // ceil(group / 8): passes over a KV head
  int per_pass;  // query heads of a pass (the last one may have fewer)
  float scale_log2;
  int* ws_cnt;
  float* ws_ml;
  float* ws_o;
  int* err;
};

template <int D>
struct Cfg {
  static constexpr int kTile = kUnit * D;      // bytes of K (or V) of a unit
  static constexpr int kStage = 2 * kTile;
  static constexpr int kKK = D / 32;           // k steps of Q K^T
  static constexpr int kDT = D / 16;           // m tiles of V^T P^T
  // Two CTAs per SM with three stages at D = 128 keep 192 KB of loads in flight per SM.
  static constexpr int kStages = D == 64 ? 5 : 3;
};

template <int D>
constexpr size_t smem_bytes(int batch) {
  return 1024 + static_cast<size_t>(kWarps) * Cfg<D>::kStages * (Cfg<D>::kStage + 8 + 16) +
         static_cast<size_t>(batch + 1) * 4;
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two 16 x 16 byte matrices, transposed: lane l receives bytes (rows 4 (l % 4) .. + 3) of columns
// l / 4 and l / 4 + 8 of the first (r0, r1) and of the second (r2, r3). Lanes 0-15 address the rows
// of the first, 16-31 those of the second.
__device__ __forceinline__ void ldmatrix_b8_trans_x2(uint32_t addr, uint32_t& r0, uint32_t& r1,
                                                     uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  return __half22float2(
      __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v), __NV_E4M3)));
}

// Nearest value with four significant bits (ties away from zero): what e4m3 keeps of x.
__device__ __forceinline__ float round4(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x00080000u) & 0xfff00000u);
}

// Byte offset o of a tile (rows of 128 bytes, 1024-byte aligned) in the 128-byte swizzle.
__device__ __forceinline__ uint32_t sw(uint32_t o) { return o ^ (((o >> 7) & 7u) << 4); }

// Token of a unit's 16-token half behind MMA row r.
__device__ __forceinline__ int row_token(int r) { return r < 8 ? r : 8 + ((r - 8) ^ 4); }

__device__ __forceinline__ int clamp_ctx(int ctx, int max_tokens) {
  return min(max(ctx, 0), max_tokens);
}

// out = sum_j w_j O_j / sum_j w_j l_j over a segment's pieces, w_j = 2^(m_j - max m).
template <typename T, int D>
__device__ __noinline__ void merge_pieces(T* dst, const float* ws_ml, const float* ws_o, int wa,
                                          int npieces, int role_a, int heads, int lane) {
  auto slot_of = [&](int j) { return static_cast<int64_t>(wa + j) * 2 + (j == 0 ? role_a : 0); };
  for (int g = 0; g < heads; ++g) {
    float M = -INFINITY;
    for (int j = lane; j < npieces; j += 32)
      M = fmaxf(M, __ldcg(ws_ml + (slot_of(j) * kHeadsPad + g) * 2));
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, x));
    float L = 0.f;
    float acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
#pragma unroll 8
    for (int j = 0; j < npieces; ++j) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(ws_ml + (slot_of(j) * kHeadsPad + g) * 2));
      const float w = ml.x == M ? 1.f : fast_exp2(ml.x - M);
      L += w * ml.y;
      const float* src = ws_o + (slot_of(j) * kHeadsPad + g) * D + lane * (D / 32);
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] += w * __ldcg(src + e);
    }
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) dst[g * D + lane * (D / 32) + e] = from_f32<T>(acc[e] * inv);
  }
}

// kWide: five to eight query heads of a pass, each part in an MMA of its own; else up to four.
template <typename T, int D, int S, bool kWide>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const Params p) {
  using C = Cfg<D>;
  constexpr int NS = C::kStages;
  constexpr int NP = kUnit / S;  // pages per unit
  constexpr int kParts = std::is_same<T, __nv_bfloat16>::value ? 2 : 3;
  constexpr int NT = kWide ? kParts : (kParts + 1) / 2;  // MMAs per step along n
  constexpr int kRows = S * D / 128;  // 128-byte rows per page tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kWarps * NS * C::kStage);
  float4* s_scale = reinterpret_cast<float4*>(bars + kWarps * NS);  // (sk0, sk1, sv0, sv1)
  int* s_uoff = reinterpret_cast<int*>(s_scale + kWarps * NS);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int B = p.batch;
  const int HV = p.hkv * p.passes;  // (KV head, pass) pairs of a request
  const int max_tokens = p.max_pages * S;
  pdl_trigger();

  // ---- exclusive prefix of unit counts over the batch ------------------------------
  {
    __shared__ int warp_tot[kWarps];
    const int per = (B + kThreads - 1) / kThreads;
    const int beg = min(tid * per, B), end = min(beg + per, B);
    auto units = [&](int i) { return (clamp_ctx(__ldg(p.ctx_lens + i), max_tokens) + kUnit - 1) / kUnit; };
    int local = 0;
    for (int i = beg; i < end; ++i) local += units(i);
    int incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    int run = incl - local;
    for (int w = 0; w < warp; ++w) run += warp_tot[w];
    for (int i = beg; i < end; ++i) {
      s_uoff[i] = run;
      run += units(i);
    }
    if (tid == kThreads - 1) s_uoff[B] = run;
  }
  const uint32_t bar0 = smem_u32(bars + warp * NS);
  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_mbar_init();
  }
  if (tid == 0) {
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  __syncthreads();

  const int NW = gridDim.x * kWarps;
  const int gw = blockIdx.x * kWarps + warp;
  const int64_t total = static_cast<int64_t>(s_uoff[B]) * HV;
  // every active warp owns at least one unit: a segment's pieces are the warps that overlap it
  const int NWe = static_cast<int>(total < NW ? total : NW);
  const bool active = gw < NWe;
  const int64_t lo = active ? total * gw / NWe : 0;
  const int64_t hi = active ? total * (gw + 1) / NWe : 0;

  auto locate = [&](int64_t pos, int& b, int& hv, int& u) {
    int l = 0, r = B - 1;
    while (l < r) {
      const int mid = (l + r + 1) >> 1;
      if (static_cast<int64_t>(s_uoff[mid]) * HV <= pos) l = mid; else r = mid - 1;
    }
    b = l;
    const int n = s_uoff[l + 1] - s_uoff[l];
    const int64_t rem = pos - static_cast<int64_t>(s_uoff[l]) * HV;
    hv = static_cast<int>(rem / n);
    u = static_cast<int>(rem - static_cast<int64_t>(hv) * n);
  };

  // Page tiles (page id * hkv + head) of stream position base + lane; -1: the unit has no second
  // page. Their scales are fetched with them.
  struct Ids {
    int t0, t1;
  };
  auto load_ids = [&](int64_t base) -> Ids {
    const int64_t pos = base + lane;
    Ids r{0, -1};
    if (pos >= hi) return r;
    int b, hv, u;
    locate(pos, b, hv, u);
    const int h = hv / p.passes;
    const int n_pages = (clamp_ctx(__ldg(p.ctx_lens + b), max_tokens) + S - 1) / S;
    const int32_t* row = p.block_tables + static_cast<int64_t>(b) * p.bt_stride + u * NP;
    auto tile = [&](int i) {
      int pid = __ldg(row + i);
      if (pid < 0 || static_cast<int64_t>(pid) >= p.num_pages) {
        record_error(p.err, PI_ERR_PAGE_RANGE);
        pid = 0;
      }
      return pid * p.hkv + h;
    };
    r.t0 = tile(0);
    if (NP == 2 && u * NP + 1 < n_pages) r.t1 = tile(1);
    return r;
  };

  const uint32_t tiles_u32 = smem_u32(tiles) + warp * NS * C::kStage;
  float4* my_scale = s_scale + warp * NS;
  int64_t pbase = lo;
  Ids id_cur = load_ids(lo), id_nxt = load_ids(lo + 32);
  // What is read above (ctx_lens and block_tables) was not written by the launch before this one.
  pdl_wait();
  float4 sc_cur, sc_nxt;
  auto load_scales = [&](const Ids& id) {
    float4 s;
    s.x = p.k_scale[id.t0];
    s.z = p.v_scale[id.t0];
    s.y = id.t1 >= 0 ? p.k_scale[id.t1] : 0.f;
    s.w = id.t1 >= 0 ? p.v_scale[id.t1] : 0.f;
    return s;
  };

  for (int b = gw; b < B; b += NW) {
    if (s_uoff[b + 1] == s_uoff[b]) {  // nothing to attend: zeros
      T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(b) * p.out_stride;
      for (int i = lane; i < p.hkv * p.group * D; i += 32) dst[i] = from_f32<T>(0.f);
    }
  }
  if (!active) return;
  sc_cur = load_scales(id_cur);
  sc_nxt = load_scales(id_nxt);

  auto issue = [&](int64_t pos, int stage) {
    if (pos - pbase >= 32) {
      pbase += 32;
      id_cur = id_nxt;
      sc_cur = sc_nxt;
      id_nxt = load_ids(pbase + 32);
      sc_nxt = load_scales(id_nxt);
    }
    const int src = static_cast<int>(pos - pbase);
    const int t0 = __shfl_sync(kFull, id_cur.t0, src);
    const int t1 = __shfl_sync(kFull, id_cur.t1, src);
    if (lane == src) my_scale[stage] = sc_cur;
    if (lane == 0) {
      const uint32_t bar = bar0 + 8 * stage;
      const uint32_t kdst = tiles_u32 + stage * C::kStage;
      const uint32_t vdst = kdst + C::kTile;
      fence_proxy_async_smem();
      mbar_arrive_expect_tx(bar, (t1 >= 0 ? 2 : 1) * 2 * S * D);
      tma_load_2d(kdst, &tmap_k, bar, 0, t0 * kRows);
      tma_load_2d(vdst, &tmap_v, bar, 0, t0 * kRows);
      if (NP == 2 && t1 >= 0) {
        tma_load_2d(kdst + S * D, &tmap_k, bar, 0, t1 * kRows);
        tma_load_2d(vdst + S * D, &tmap_v, bar, 0, t1 * kRows);
      }
    }
  };

  int64_t issued = lo;
  for (int s = 0; s < NS && issued < hi; ++s, ++issued) issue(issued, s);

  const int gid = lane >> 2;
  const int tig = lane & 3;
  // K: matrix lane / 8, row lane % 8: rows 0-7 / 8-15, bytes 0-15 / 16-31 of each 32
  const int k_tok = row_token((lane & 7) + 8 * ((lane >> 3) & 1));
  const uint32_t k_off = static_cast<uint32_t>(k_tok * D + 16 * (lane >> 4));
  // V: row i = lane % 16 of matrix lane / 16 is the token of k slot i
  const int vi = lane & 15;
  const int v_tok = row_token(2 * (vi >> 2) + ((vi & 3) >> 1) + 8 * (vi & 1));
  const uint32_t v_off = static_cast<uint32_t>((16 * (lane >> 4) + v_tok) * D);
  const int r0_tok = gid, r1_tok = 8 + (gid ^ 4);  // tokens of accumulator rows gid, gid + 8
  const int head_a = kWide ? 2 * tig : (2 * tig) & 3;  // heads of accumulator columns
  const bool first_part = tig < 2;

  uint32_t qf[NT][C::kKK][2];
  float f0, f1;  // 2^-k scale log2(e) of the two heads
  // Query rows of (request b, head pass hv) as e4m3 parts; heads beyond the pass are zero.
  auto load_q = [&](int b, int hv) {
    const int h = hv / p.passes, pass = hv - h * p.passes;
    const int first = pass * p.per_pass;
    const int heads = min(p.per_pass, p.group - first);
    const int my = kWide ? gid : gid & 3;
    const T* row = static_cast<const T*>(p.q) + static_cast<int64_t>(b) * p.q_stride +
                   static_cast<int64_t>(h * p.group + first + my) * D + 4 * tig;
    float x[C::kKK][8];
    float amax = 0.f;
#pragma unroll
    for (int kk = 0; kk < C::kKK; ++kk) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint2 w = make_uint2(0u, 0u);
        if (my < heads) w = __ldg(reinterpret_cast<const uint2*>(row + 32 * kk + 16 * half));
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[kk][4 * half + i] = to_f32(e[i]);
          amax = fmaxf(amax, fabsf(x[kk][4 * half + i]));
        }
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
    // largest element into [128, 256); an infinity makes the row NaN, as inf - inf would
    const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23), 8), 254);
    const float up = amax < INFINITY ? __uint_as_float(static_cast<uint32_t>(261 - e) << 23)
                                     : __uint_as_float(0x7fffffffu);
    const float down = __uint_as_float(static_cast<uint32_t>(e - 7) << 23);
#pragma unroll
    for (int kk = 0; kk < C::kKK; ++kk) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t part[kParts];
        float r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = x[kk][4 * half + i] * up;
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          const uint32_t a = e4m3x2(r[0], r[1]), c = e4m3x2(r[2], r[3]);
          part[j] = a | (c << 16);
          const float2 fa = from_e4m3x2(a), fc = from_e4m3x2(c);
          r[0] -= fa.x;
          r[1] -= fa.y;
          r[2] -= fc.x;
          r[3] -= fc.y;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (kWide) qf[j][kk][half] = part[j];
          else qf[j][kk][half] = gid < 4 ? part[2 * j] : (2 * j + 1 < kParts ? part[2 * j + 1 < kParts ? 2 * j + 1 : 0] : 0u);
        }
      }
    }
    f0 = __shfl_sync(kFull, down, 4 * head_a) * p.scale_log2;
    f1 = __shfl_sync(kFull, down, 4 * (head_a + 1)) * p.scale_log2;
  };

  float o[C::kDT][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  int cb, chv, cu;
  locate(lo, cb, chv, cu);
  int cn = s_uoff[cb + 1] - s_uoff[cb];
  int cctx = clamp_ctx(__ldg(p.ctx_lens + cb), max_tokens);
  int64_t piece_start = lo;
  bool fresh = true, failed = false;
  int64_t pos = lo;
  int k = 0;

  auto finalize = [&](int64_t piece_end) {
    float t0 = l0, t1 = l1;
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      t0 += __shfl_xor_sync(kFull, t0, x);
      t1 += __shfl_xor_sync(kFull, t1, x);
    }
    if constexpr (!kWide) {  // part 2's share of O sits in columns 4-7
#pragma unroll
      for (int dt = 0; dt < C::kDT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[dt][i] += __shfl_xor_sync(kFull, o[dt][i], 2);
    }
    const int h = chv / p.passes, pass = chv - h * p.passes;
    const int first = pass * p.per_pass;
    const int heads = min(p.per_pass, p.group - first);
    const int64_t seg_start = static_cast<int64_t>(s_uoff[cb]) * HV + static_cast<int64_t>(chv) * cn;
    const int64_t seg_end = seg_start + cn;
    T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(cb) * p.out_stride +
             static_cast<int64_t>(h * p.group + first) * D;
    const bool mine = kWide || first_part;
    const int g0 = head_a, g1 = head_a + 1;
    if (piece_start == seg_start && piece_end == seg_end) {
      const float i0 = 1.f / t0, i1 = 1.f / t1;
#pragma unroll
      for (int dt = 0; dt < C::kDT; ++dt) {
        const int d = 16 * dt + gid;
        if (mine && g0 < heads) {
          dst[g0 * D + d] = from_f32<T>(o[dt][0] * i0);
          dst[g0 * D + d + 8] = from_f32<T>(o[dt][2] * i0);
        }
        if (mine && g1 < heads) {
          dst[g1 * D + d] = from_f32<T>(o[dt][1] * i1);
          dst[g1 * D + d + 8] = from_f32<T>(o[dt][3] * i1);
        }
      }
      return;
    }
    const int role = piece_start == lo ? 0 : 1;
    const int64_t slot = static_cast<int64_t>(gw) * 2 + role;
    float* wo = p.ws_o + slot * kHeadsPad * D;
#pragma unroll
    for (int dt = 0; dt < C::kDT; ++dt) {
      const int d = 16 * dt + gid;
      if (mine && g0 < heads) {
        wo[g0 * D + d] = o[dt][0];
        wo[g0 * D + d + 8] = o[dt][2];
      }
      if (mine && g1 < heads) {
        wo[g1 * D + d] = o[dt][1];
        wo[g1 * D + d + 8] = o[dt][3];
      }
    }
    if (gid == 0 && mine) {
      float* wml = p.ws_ml + slot * kHeadsPad * 2;
      wml[g0 * 2] = m0;
      wml[g0 * 2 + 1] = t0;
      wml[g1 * 2] = m1;
      wml[g1 * 2 + 1] = t1;
    }
    __threadfence();
    __syncwarp();
    int* cnt = p.ws_cnt + cb * HV + chv;
    int old = 0;
    if (lane == 0) old = atomicAdd(cnt, 1);
    old = __shfl_sync(kFull, old, 0);
    const int wa = static_cast<int>(((seg_start + 1) * NWe - 1) / total);
    const int wb = static_cast<int>((seg_end * NWe - 1) / total);
    const int npieces = wb - wa + 1;
    if (old != npieces - 1) return;
    __threadfence();
    const int role_a = (total * wa / NWe == seg_start) ? 0 : 1;
    merge_pieces<T, D>(dst, p.ws_ml, p.ws_o, wa, npieces, role_a, heads, lane);
    if (lane == 0) *cnt = 0;
  };

  while (pos < hi) {
    if (fresh) {
      load_q(cb, chv);
#pragma unroll
      for (int dt = 0; dt < C::kDT; ++dt) o[dt][0] = o[dt][1] = o[dt][2] = o[dt][3] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
      piece_start = pos;
      fresh = false;
    }
    const int stage = k % NS;
    if (!mbar_wait_bounded(bar0 + 8 * stage, static_cast<uint32_t>((k / NS) & 1))) {
      if (lane == 0) record_error(p.err, PI_ERR_TIMEOUT);
      failed = true;
      break;
    }
    __syncwarp();
    const uint32_t ktile = tiles_u32 + stage * C::kStage;
    const uint32_t vtile = ktile + C::kTile;
    const float4 scales = my_scale[stage];
    const int valid = min(kUnit, cctx - cu * kUnit);
    if (valid < kUnit) {
      // V rows past the context may hold anything, NaN included, and a weight of zero does not
      // hide it: clear them.
      uint8_t* vt = tiles + (warp * NS + stage) * C::kStage + C::kTile;
      for (int c = valid * (D / 16) + lane; c < kUnit * (D / 16); c += 32)
        *reinterpret_cast<uint4*>(vt + sw(16 * c)) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }

    // S^T in base-2 units, masked
    float s[2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < C::kKK; ++kk) {
        uint32_t a0, a1, a2, a3;
        ldmatrix_x4(ktile + sw(k_off + 16 * mt * D + 32 * kk), a0, a1, a2, a3);
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_e4m3(c, a0, a1, a2, a3, qf[j][kk][0], qf[j][kk][1]);
      }
      if constexpr (!kWide) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += __shfl_xor_sync(kFull, c[i], 2);
      }
      const float sk = (NP == 2 && mt == 1) ? scales.y : scales.x;
      const float a = f0 * sk, b = f1 * sk;
      const bool v0 = 16 * mt + r0_tok < valid, v1 = 16 * mt + r1_tok < valid;
      s[mt][0] = v0 ? c[0] * a : -INFINITY;
      s[mt][1] = v0 ? c[1] * b : -INFINITY;
      s[mt][2] = v1 ? c[2] * a : -INFINITY;
      s[mt][3] = v1 ? c[3] * b : -INFINITY;
    }
    float u0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
    float u1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      u0 = fmaxf(u0, __shfl_xor_sync(kFull, u0, x));
      u1 = fmaxf(u1, __shfl_xor_sync(kFull, u1, x));
    }
    const float n0 = fmaxf(m0, u0), n1 = fmaxf(m1, u1);
    const float al0 = fast_exp2(m0 - n0), al1 = fast_exp2(m1 - n1);
    const float be0 = fast_exp2(u0 - n0), be1 = fast_exp2(u1 - n1);
    m0 = n0;
    m1 = n1;
    // P relative to the unit's maximum (times 256) and to its larger V scale
    float sv = scales.z, w0 = 1.f, w1 = 1.f;
    if (NP == 2) {
      sv = fmaxf(scales.z, scales.w);
      const float ratio = sv > 0.f ? fminf(scales.z, scales.w) / sv : 0.f;
      w0 = scales.z == sv ? 1.f : ratio;
      w1 = scales.w == sv ? 1.f : ratio;
    }
    uint32_t pb[NT][2];
    float q0 = 0.f, q1 = 0.f;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      float e[4];
      e[0] = fast_exp2(s[mt][0] - u0 + 8.f);
      e[1] = fast_exp2(s[mt][1] - u1 + 8.f);
      e[2] = fast_exp2(s[mt][2] - u0 + 8.f);
      e[3] = fast_exp2(s[mt][3] - u1 + 8.f);
      q0 += e[0] + e[2];
      q1 += e[1] + e[3];
      float part[kParts][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float r = NP == 2 ? e[i] * (mt ? w1 : w0) : e[i];
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          part[j][i] = j + 1 < kParts ? round4(r) : r;
          r -= part[j][i];
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kWide) x[i] = part[j][i];
          else x[i] = first_part ? part[2 * j][i] : (2 * j + 1 < kParts ? part[2 * j + 1 < kParts ? 2 * j + 1 : 0][i] : 0.f);
        }
        pb[j][mt] = movmatrix_trans(e4m3x2(x[0], x[2]) | (e4m3x2(x[1], x[3]) << 16));
      }
    }
    l0 = l0 * al0 + be0 * q0;
    l1 = l1 * al1 + be1 * q1;
    const float bs0 = be0 * sv, bs1 = be1 * sv;
#pragma unroll
    for (int dt = 0; dt < C::kDT; ++dt) {
      uint32_t a0, a1, a2, a3;
      ldmatrix_b8_trans_x2(vtile + sw(v_off + 16 * dt), a0, a1, a2, a3);
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NT; ++j) mma_e4m3(c, a0, a1, a2, a3, pb[j][0], pb[j][1]);
      o[dt][0] = o[dt][0] * al0 + c[0] * bs0;
      o[dt][1] = o[dt][1] * al1 + c[1] * bs1;
      o[dt][2] = o[dt][2] * al0 + c[2] * bs0;
      o[dt][3] = o[dt][3] * al1 + c[3] * bs1;
    }
    __syncwarp();
    if (issued < hi) {
      issue(issued, stage);
      ++issued;
    }
    ++k;
    ++pos;
    if (++cu == cn) {
      finalize(pos);
      if (pos < hi) {
        cu = 0;
        if (++chv == HV) {
          chv = 0;
          do { ++cb; } while (cb < B && s_uoff[cb + 1] == s_uoff[cb]);
        }
        cn = s_uoff[cb + 1] - s_uoff[cb];
        cctx = clamp_ctx(__ldg(p.ctx_lens + cb), max_tokens);
        fresh = true;
      }
    } else if (pos == hi) {
      finalize(pos);
    }
  }
  if (failed) {  // loads in flight land before the shared memory is released
    for (int64_t j = k; j < issued - lo; ++j)
      mbar_wait_bounded(bar0 + 8 * static_cast<int>(j % NS), static_cast<uint32_t>((j / NS) & 1));
  }
}

// ---------------------------------------------------------------------------------
// Generic kernel: one CTA per (request, query head), four warps over the tokens.
// ---------------------------------------------------------------------------------

constexpr int kGenericMaxD = 256;

__device__ __forceinline__ float e4m3_value(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

template <typename T>
__global__ void __launch_bounds__(128)
    decode_q8_generic_kernel(const Params p, const uint8_t* k_pool, const uint8_t* v_pool, int D, int S) {
  pdl_trigger();
  pdl_wait();
  const int hq = blockIdx.x;
  const int h = hq / p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float q_s[kGenericMaxD];
  __shared__ float w_m[4], w_l[4];
  __shared__ float w_acc[4][kGenericMaxD];
  for (int b = blockIdx.y; b < p.batch; b += gridDim.y) {
    const T* qrow = static_cast<const T*>(p.q) + static_cast<int64_t>(b) * p.q_stride +
                    static_cast<int64_t>(hq) * D;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += blockDim.x) q_s[d] = to_f32(qrow[d]) * p.scale_log2;
    __syncthreads();
    const int64_t most = static_cast<int64_t>(p.max_pages) * S;
    const int ctx = clamp_ctx(__ldg(p.ctx_lens + b), most > 0x7fffffff ? 0x7fffffff : static_cast<int>(most));
    float m = -INFINITY, l = 0.f;
    float acc[kGenericMaxD / 32];
#pragma unroll
    for (int e = 0; e < kGenericMaxD / 32; ++e) acc[e] = 0.f;
    for (int64_t t0 = 32 * warp; t0 < ctx; t0 += 128) {  // lane = token
      const int64_t t = t0 + lane;
      float sc = -INFINITY, sv = 0.f;
      int64_t row = -1;
      if (t < ctx) {
        const int pid = __ldg(p.block_tables + static_cast<int64_t>(b) * p.bt_stride + t / S);
        if (pid < 0 || pid >= p.num_pages) {
          record_error(p.err, PI_ERR_PAGE_RANGE);
        } else {
          const int64_t block = static_cast<int64_t>(pid) * p.hkv + h;
          row = (block * S + t % S) * D;
          float dot = 0.f;
          for (int d = 0; d < D; ++d) dot += q_s[d] * e4m3_value(k_pool[row + d]);
          sc = dot * p.k_scale[block];
          sv = p.v_scale[block];
        }
      }
      float mx = sc;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, x));
      const float mn = fmaxf(m, mx);
      const float pt = row < 0 ? 0.f : exp2f(sc - mn);
      const float al = m == mn ? 1.f : exp2f(m - mn);
      float ps = pt;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) ps += __shfl_xor_sync(kFull, ps, x);
      l = l * al + ps;
      m = mn;
#pragma unroll
      for (int e = 0; e < kGenericMaxD / 32; ++e) acc[e] *= al;
      for (int tt = 0; tt < 32; ++tt) {
        const int64_t r = __shfl_sync(kFull, row, tt);
        const float w = __shfl_sync(kFull, pt * sv, tt);
        if (r < 0) continue;
#pragma unroll
        for (int e = 0; e < kGenericMaxD / 32; ++e) {
          const int d = lane + 32 * e;
          if (d < D) acc[e] += w * e4m3_value(v_pool[r + d]);
        }
      }
    }
    if (lane == 0) {
      w_m[warp] = m;
      w_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < kGenericMaxD / 32; ++e)
      if (lane + 32 * e < D) w_acc[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    const float M = fmaxf(fmaxf(w_m[0], w_m[1]), fmaxf(w_m[2], w_m[3]));
    float L = 0.f, wt[4];
    for (int w = 0; w < 4; ++w) {
      wt[w] = w_l[w] == 0.f ? 0.f : (w_m[w] == M ? 1.f : exp2f(w_m[w] - M));
      L += wt[w] * w_l[w];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* orow = static_cast<T*>(p.out) + static_cast<int64_t>(b) * p.out_stride + static_cast<int64_t>(hq) * D;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
      float v = 0.f;
      for (int w = 0; w < 4; ++w) v += wt[w] * w_acc[w][d];
      orow[d] = from_f32<T>(v * inv);
    }
  }
}

// ---------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------

// A pool as rows of 128 bytes; a page tile is one box.
bool pool_map(CUtensorMap* m, const void* base, uint64_t rows, int box_rows) {
  auto encode = attn::get_encode();
  if (!encode) return false;
  cuuint64_t dims[2] = {128, rows};
  cuuint64_t strides[1] = {128};
  cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Layout {
  size_t ml_off, o_off, total;
};
inline size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
// [arrival counters | partial (max, sum) | partial O]; the counters have one place for every
// shape, so zeroed once they stay zero between launches.
constexpr size_t kCounterBytes = static_cast<size_t>(kMaxSegments) * sizeof(int);
Layout ws_layout(int head_dim, int sms) {
  Layout L;
  const size_t slots = static_cast<size_t>(sms) * kMaxCtasPerSm * kWarps * 2;
  L.ml_off = align256(kCounterBytes);
  L.o_off = L.ml_off + align256(slots * kHeadsPad * 2 * sizeof(float));
  L.total = L.o_off + align256(slots * kHeadsPad * static_cast<size_t>(head_dim) * sizeof(float));
  return L;
}

bool fast_shape(int dtype, int batch, int hkv, int group, int D, int S, int64_t pages, int max_pages) {
  return (dtype == PI_DTYPE_BF16 || dtype == PI_DTYPE_F16) && (D == 64 || D == 128 || D == 256) &&
         (S == 16 || S == 32) && batch <= kMaxBatch &&
         static_cast<int64_t>(batch) * hkv * ((group + 7) / 8) <= kMaxSegments &&
         pages * hkv * (S * D / 128) <= 0x7fffffff && pages * hkv <= 0x7fffffff && pages > 0 &&
         static_cast<int64_t>(max_pages) * S <= 0x7fffffff - kUnit &&
         // positions of the unit stream times warps stay far inside 64 bits, counts inside 32
         static_cast<int64_t>(batch) * ((static_cast<int64_t>(max_pages) * S + kUnit - 1) / kUnit) <= 0x7fffffff;
}

template <typename T, int D, int S, bool kWide>
int launch(const Params& p, const void* k_pool, const void* v_pool, cudaStream_t stream) {
  auto kern = decode_q8_kernel<T, D, S, kWide>;
  static std::atomic<int> configured[64];  // CTAs per SM + 1, per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return PI_ERR_CUDA;
  if (dev < 0 || dev >= 64) return PI_ERR_UNSUPPORTED;
  const size_t smem = smem_bytes<D>(p.batch);
  if (configured[dev].load(std::memory_order_acquire) == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem_bytes<D>(kMaxBatch))) != cudaSuccess)
      return PI_ERR_CUDA;
    configured[dev].store(1, std::memory_order_release);
  }
  // two CTAs share an SM while the prefix table leaves room for both
  const int per_sm = D <= 128 && 2 * (smem + 1024) <= 228 * 1024 ? 2 : 1;
  const uint64_t rows = static_cast<uint64_t>(p.num_pages) * p.hkv * (S * D / 128);
  CUtensorMap tk, tv;
  if (!pool_map(&tk, k_pool, rows, S * D / 128) || !pool_map(&tv, v_pool, rows, S * D / 128))
    return PI_ERR_CUDA;
  return cuda_status(launch_kernel(kern, dim3(device_sm_count() * per_sm), dim3(kThreads), smem, stream,
                                   tk, tv, p));
}

}  // namespace q8
}  // namespace pi

extern "C" size_t pi_paged_decode_attn_q8_workspace_bytes(int head_dim) {
  if (head_dim <= 0) return 0;
  return pi::q8::ws_layout(head_dim, pi::device_sm_count()).total;
}

extern "C" size_t pi_paged_decode_attn_q8_ws_zero_bytes(void) {
  return pi::q8::align256(pi::q8::kCounterBytes);
}

extern "C" int pi_paged_decode_attn_q8(void* out, const void* q, const void* k_pool,
                                       const void* v_pool, const float* k_scale,
                                       const float* v_scale, const int32_t* block_tables,
                                       int64_t bt_stride, int max_pages, const int32_t* ctx_lens,
                                       int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                       int page_size, int64_t num_pages, float scale, int dtype,
                                       int64_t q_stride, int64_t out_stride, void* workspace,
                                       size_t workspace_bytes, int* err, cudaStream_t stream) {
  using namespace pi;
  const int eb = elem_bytes_of(dtype);
  if (eb == 0) return PI_ERR_UNSUPPORTED;
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || page_size <= 0 ||
      num_pages < 0 || max_pages < 0 || bt_stride < 0 || num_q_heads % num_kv_heads != 0)
    return PI_ERR_BAD_SHAPE;
  const int64_t row = static_cast<int64_t>(num_q_heads) * head_dim;
  if (q_stride < row || out_stride < row || row > 0x7fffffff) return PI_ERR_BAD_SHAPE;
  if (head_dim > q8::kGenericMaxD) return PI_ERR_UNSUPPORTED;
  if (batch == 0) return PI_OK;
  if (!out || !q || !k_pool || !v_pool || !k_scale || !v_scale || !ctx_lens ||
      (max_pages > 0 && !block_tables))
    return PI_ERR_NULL_POINTER;
  if (!aligned(block_tables, 4) || !aligned(ctx_lens, 4) || !aligned(k_scale, 4) ||
      !aligned(v_scale, 4) || !aligned(q, eb) || !aligned(out, eb))
    return PI_ERR_MISALIGNED;
  const int group = num_q_heads / num_kv_heads;
  q8::Params p;
  p.out = out;
  p.q = q;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.ctx_lens = ctx_lens;
  p.bt_stride = bt_stride;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.num_pages = num_pages;
  p.batch = batch;
  p.max_pages = num_pages > 0 ? max_pages : 0;
  p.hkv = num_kv_heads;
  p.group = group;
  p.passes = (group + 7) / 8;
  p.per_pass = (group + p.passes - 1) / p.passes;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.ws_cnt = nullptr;
  p.ws_ml = p.ws_o = nullptr;
  p.err = err;
  const bool fast = q8::fast_shape(dtype, batch, num_kv_heads, group, head_dim, page_size, num_pages,
                                   max_pages) &&
                    aligned(k_pool, 16) && aligned(v_pool, 16) && aligned(q, 8) && q_stride % 4 == 0;
  if (fast) {
    const q8::Layout L = q8::ws_layout(head_dim, device_sm_count());
    if (workspace == nullptr || workspace_bytes < L.total) return PI_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return PI_ERR_MISALIGNED;
    char* ws = static_cast<char*>(workspace);
    p.ws_cnt = reinterpret_cast<int*>(ws);
    p.ws_ml = reinterpret_cast<float*>(ws + L.ml_off);
    p.ws_o = reinterpret_cast<float*>(ws + L.o_off);
#define PI_Q8(T, D, S)                                                                         \
  if (head_dim == D && page_size == S)                                                         \
    return p.per_pass > 4 ? q8::launch<T, D, S, true>(p, k_pool, v_pool, stream)               \
                          : q8::launch<T, D, S, false>(p, k_pool, v_pool, stream);
#define PI_Q8_ALL(T) PI_Q8(T, 64, 16) PI_Q8(T, 64, 32) PI_Q8(T, 128, 16) PI_Q8(T, 128, 32) \
                     PI_Q8(T, 256, 16) PI_Q8(T, 256, 32)
    if (dtype == PI_DTYPE_BF16) { PI_Q8_ALL(__nv_bfloat16) } else { PI_Q8_ALL(__half) }
#undef PI_Q8_ALL
#undef PI_Q8
  }
  const dim3 grid(num_q_heads, batch < 65535 ? batch : 65535);
  const uint8_t* kp = static_cast<const uint8_t*>(k_pool);
  const uint8_t* vp = static_cast<const uint8_t*>(v_pool);
  switch (dtype) {
    case PI_DTYPE_F32:
      return cuda_status(launch_kernel(q8::decode_q8_generic_kernel<float>, grid, dim3(128), 0, stream, p, kp, vp, head_dim, page_size));
    case PI_DTYPE_BF16:
      return cuda_status(launch_kernel(q8::decode_q8_generic_kernel<__nv_bfloat16>, grid, dim3(128), 0, stream, p, kp, vp, head_dim, page_size));
    default:
      return cuda_status(launch_kernel(q8::decode_q8_generic_kernel<__half>, grid, dim3(128), 0, stream, p, kp, vp, head_dim, page_size));
  }
}
