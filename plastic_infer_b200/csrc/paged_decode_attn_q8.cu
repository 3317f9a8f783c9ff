// Batched paged GQA decode attention over an 8-bit cache: K and V pools of e4m3 values with one
// scale per (page, KV head), one query token per request.
//
//   out[b, hq] = sum_t p_t sv(t) V[t] / sum_t p_t,   p_t = exp(scale * sk(t) q . K[t] - max)
//
// What bounds it: K and V once, HBM. At half the bytes of a 16-bit cache the arithmetic per byte
// doubles, and mma.sync has no 8-bit float form of its own on sm_100a: m16n8k32 e4m3 measured 0.13
// per clock and SM with fresh operands, against 0.30 for the 16-bit m16n8k16 it is put together
// from. So a unit's values are widened once, in registers, by cvt.rn.f16x2.e4m3x2 (1.2 per clock
// and SM; every e4m3 value is an f16 value), and both products are f16 MMAs with fp32 sums:
//   q 2^k in f16: exact for bf16 and f16 down to 2^-21 of the row's largest element, which k
//   brings into [128, 256);
//   P in f16, relative to the unit's own maximum and to its larger V scale, times 256: half a step is
//   2^-11 of each weight, or 2^-33 of the unit's largest. A page whose V scale is 2^-k of its
//   neighbour's in the unit has its weights k bits lower, and loses what falls below.
// (q and P in e4m3 parts, two for bf16 and three for f16, with K and V as they are: 112.6 us for the 64
// requests below.)
//
// A step of a warp is a unit of 32 tokens (two pages of 16, or one of 32):
//   S^T[tokens, heads] = K[tokens, D] . Q^T           A = K by ldmatrix, widened
//   softmax of the unit against its own maximum, then
//   O^T[D, heads] = alpha O^T + beta (V^T[D, tokens] . P^T[tokens, heads])
//                                                     A = V^T by ldmatrix .b8 transposed, widened
// beta = 2^(max_unit - max) sv. A lane's four bytes of K or V become the two k pairs of a fragment;
// the order of the elements along k that this implies is put into Q's loads, and for V into the
// row addresses of its ldmatrix. The MMA rows 8..15 are tokens 12..15, 8..11, which keeps both
// K's and V's ldmatrix free of bank conflicts in the 128-byte swizzle.
//
// Work: the stream of units over (request, KV head) is cut into equal ranges, one per resident
// warp, each with its own ring of TMA stages; pieces of a cut (request, head) are merged by the
// last warp to finish one (the counters return to zero). More than eight query heads per KV
// head run as several passes over it.
//
// Measured on B200 (32 query and 8 KV heads of 128): 64 requests of 512-8192 tokens, 572 MB, in
// 103 us, 5.5 TB/s, 0.84 of the measured copy rate; 8 of 32k (f16, pages of 32) in 96 us, 0.82; 128 of
// 200-4096 with 8 query heads per KV head, 286 MB, in 62 us, 0.70. What is left: some 4 us until the
// first loads are out, and the spread of the warps' ends (the same SMs are up to 15 % late in every
// launch). One CTA per SM with loader warps, items from a queue and a quarter of the stream handed
// out dynamically evened the ends out, but its waits for items and partial sums cost more than
// that: 129 us for the first.
//
// Generic kernel (fp32 queries, other head sizes and pages): one CTA per (request, query head).
#include <atomic>
#include <type_traits>

#include <cuda_fp8.h>
#include <cudaTypedefs.h>

#include "pi_common.cuh"
#include "q8_split.cuh"

namespace pi {
namespace attn {
// paged_decode_attn.cu
bool encode_tiled(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                  const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);
}  // namespace attn

namespace q8 {

constexpr int kWarps = 4;  // per CTA, each an independent consumer
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 32;            // tokens per step
constexpr int kMaxBatch = 4096;
constexpr int kMaxSegments = kAttnSegments;
constexpr int kMaxCtasPerSm = 2;
constexpr int kMaxTiles = 2;          // tiles of eight query rows per pass
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
  int group;     // query heads per KV head
  int rows;      // query rows of a request per KV head: group, or q_len * group
  int passes;    // over a KV head's rows
  int per_pass;  // rows of a pass (the last one may have fewer)
  // One request's several query tokens (ctx_lens null, batch 1): row r is token r / group, at
  // position q_start + r / group; causal ones see no key behind them.
  int q_len, kv_len, q_start, causal;
  int merge_later;  // pieces are left to merge_kernel
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
  static constexpr int kKK = D / 16;           // k steps of Q K^T
  static constexpr int kDT = D / 16;           // m tiles of V^T P^T
  // 128 KB of loads in flight per SM (two CTAs; one at D = 256). More only lengthens the queue in
  // front of HBM, where every small access waits too, and pulls the SMs apart: with three stages
  // at D = 128 (192 KB) 64 requests of 512-8192 tokens took 114 us against 105, 8 of 32k 104
  // against 96.
  static constexpr int kStages = D == 64 ? 4 : 2;
  static_assert(kWarps * kStages % 2 == 0, "the stages' scales follow their barriers, 16-byte aligned");
};

template <int D>
constexpr size_t smem_bytes(int batch) {
  return 1024 + static_cast<size_t>(kWarps) * Cfg<D>::kStages * (Cfg<D>::kStage + 8 + 16) +
         static_cast<size_t>(2 * batch + 1) * 4;
}

// (not volatile: pure functions of their operands, free to be scheduled)
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Four e4m3 values as two f16 pairs (exact).
__device__ __forceinline__ void widen(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

// Paired fp32 multiply and fused multiply-add.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
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

// Byte offset o of a tile (rows of 128 bytes, 1024-byte aligned) in the 128-byte swizzle. Linear
// over xor, so sw(lane's part) ^ sw(constant) addresses the sum of two disjoint offsets.
__host__ __device__ constexpr uint32_t sw(uint32_t o) { return o ^ (((o >> 7) & 7u) << 4); }

// Token of a unit's 16-token half behind MMA row r.
__device__ __forceinline__ int row_token(int r) { return r < 8 ? r : 8 + ((r - 8) ^ 4); }

__device__ __forceinline__ int clamp_ctx(int ctx, int max_tokens) {
  return min(max(ctx, 0), max_tokens);
}

// Where the query rows of one (request, KV head) pass are in q and out.
template <typename T>
struct Rows {
  T* base;
  int64_t tok_stride;
  int group, first;
  bool chunk;
  __device__ __forceinline__ T* at(int c, int D) const {
    if (!chunk) return base + static_cast<int64_t>(first + c) * D;
    const int t = (first + c) / group;
    return base + t * tok_stride + static_cast<int64_t>(first + c - t * group) * D;
  }
};

// out = sum_j w_j O_j / sum_j w_j l_j over the np pieces of a segment, w_j = 2^(m_j - max m). One
// warp, often at the launch's end, so latency counts: all heads at once in float4 columns, several
// pieces' loads in flight before any is used.
template <typename T, int D, int kPad>
__device__ __noinline__ void merge_pieces(const Rows<T> dst, const float* ml0, const float* o0, int wa,
                                          int np, int role_a, int rows, int lane) {
  for (int h0 = 0; h0 < rows; h0 += 8) {
    const float* ws_ml = ml0 + 2 * h0;
    const float* ws_o = o0 + h0 * D;
    const int heads = min(rows - h0, 8);
    auto slot_of = [&](int j) { return static_cast<int64_t>(wa + j) * 2 + (j == 0 ? role_a : 0); };
    constexpr int E = 8 * D / 128;          // float4 columns per lane, eight rows
    constexpr int kPerHead = D / 4;
    constexpr int kCols = E < 4 ? E : 4;    // columns at a time
    constexpr int kPieces = 4;              // pieces at a time
    const int n4 = heads * kPerHead;
    const int hd = min(lane & 7, heads - 1);
    const float2* mls = reinterpret_cast<const float2*>(ws_ml) + hd;
    // maximum and sum of head lane % 8, pieces lane / 8 of every four
    float top = -INFINITY;
#pragma unroll 4
    for (int j = lane >> 3; j < np; j += 4) top = fmaxf(top, __ldcg(mls + slot_of(j) * kPad).x);
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 8));
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 16));
    for (int e0 = 0; 32 * e0 < n4; e0 += kCols) {
      float4 acc[kCols];
      float sum[kCols], tops[kCols];
#pragma unroll
      for (int e = 0; e < kCols; ++e) {
        acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        sum[e] = 0.f;
        tops[e] = __shfl_sync(kFull, top, (min(lane + 32 * (e0 + e), n4 - 1) / kPerHead) & 7);
      }
      for (int j0 = 0; j0 < np; j0 += kPieces) {
        float4 v[kPieces][kCols];
        float2 ml[kPieces][kCols];
#pragma unroll
        for (int jj = 0; jj < kPieces; ++jj) {
          const int64_t s = slot_of(min(j0 + jj, np - 1));
#pragma unroll
          for (int e = 0; e < kCols; ++e) {  // (a branch here would put the loads one after another)
            const int c = min(lane + 32 * (e0 + e), n4 - 1);
            v[jj][e] = __ldcg(reinterpret_cast<const float4*>(ws_o + s * kPad * D) + c);
            ml[jj][e] = __ldcg(reinterpret_cast<const float2*>(ws_ml) + s * kPad + c / kPerHead);
          }
        }
#pragma unroll
        for (int jj = 0; jj < kPieces; ++jj) {
#pragma unroll
          for (int e = 0; e < kCols; ++e) {
            float a = ml[jj][e].x == tops[e] ? 1.f : fast_exp2(ml[jj][e].x - tops[e]);
            if (j0 + jj >= np) a = 0.f;
            sum[e] += a * ml[jj][e].y;
            acc[e].x += a * v[jj][e].x;
            acc[e].y += a * v[jj][e].y;
            acc[e].z += a * v[jj][e].z;
            acc[e].w += a * v[jj][e].w;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < kCols; ++e) {
        const int c = lane + 32 * (e0 + e);
        if (c < n4) {
          const float inv = 1.f / sum[e];
          T* o = dst.at(h0 + c / kPerHead, D) + 4 * (c % kPerHead);
          o[0] = from_f32<T>(acc[e].x * inv);
          o[1] = from_f32<T>(acc[e].y * inv);
          o[2] = from_f32<T>(acc[e].z * inv);
          o[3] = from_f32<T>(acc[e].w * inv);
        }
      }
    }
  }
}

// The arrivals of a warp whose wait expired (one lane; noinline: never on the way of a sound launch).
__device__ __noinline__ void give_up(const Split& s, const int* uoff, int requests, int HV, int warp, int64_t pos,
                                     int* counters) {
  abandon(s, uoff, requests, HV, warp, pos, [&](int segment, int pieces) {
    if (atomicAdd(counters + segment, 1) == pieces - 1) counters[segment] = 0;
  });
}

// Few segments have many pieces each: one warp that merges 150 of them after the stream's end takes
// longer than the stream (8000 tokens of 8 KV heads: 88 us). Up to kMergeSegments segments a second
// launch merges instead, a CTA to a query row, its warps side by side over the pieces; beyond that
// a segment has some eight pieces at most, and the launch costs more than it saves.
constexpr int kMergeSegments = 148;

template <typename T, int D, int kPad, bool kChunk>
__global__ void __launch_bounds__(128) merge_kernel(const Params p, int S, int NW) {
  pdl_trigger();
  pdl_wait();
  const int HV = p.hkv * p.passes;
  const int seg = blockIdx.x / p.per_pass, row = blockIdx.x - seg * p.per_pass;
  const int b = seg / HV, hv = seg - b * HV;
  const int n = min(p.per_pass, p.rows - hv % p.passes * p.per_pass);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int s_units[kMergeSegments];
  __shared__ float s_m[4], s_l[4];
  __shared__ float s_o[4][D];
  for (int i = threadIdx.x; i < p.batch; i += 128) {
    const int ctx = clamp_ctx(kChunk ? (p.causal ? min(p.kv_len, p.q_start + p.q_len) : p.kv_len)
                                     : __ldg(p.ctx_lens + i), p.max_pages * S);
    s_units[i] = (ctx + kUnit - 1) / kUnit;
  }
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < p.batch; ++i) {
    if (i < b) before += s_units[i];
    all += s_units[i];
  }
  const int64_t total = static_cast<int64_t>(all) * HV;
  const int cn = s_units[b];
  if (cn == 0 || row >= n) return;
  const Split split{total, active_warps(total, NW)};
  const int64_t start = static_cast<int64_t>(before) * HV + static_cast<int64_t>(hv) * cn;
  const int wa = split.owner(start), wb = split.owner(start + cn - 1);
  if (wa == wb) return;  // one warp had it all and has written it
  const int role_a = split.first(wa) == start ? 0 : 1;
  const int np = wb - wa + 1;
  auto at = [&](int j) { return (static_cast<int64_t>(wa + j) * 2 + (j == 0 ? role_a : 0)) * kPad + row; };
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
  float top = -INFINITY;
  for (int j = threadIdx.x; j < np; j += 128) top = fmaxf(top, __ldcg(ml + at(j)).x);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, x));
  if (lane == 0) s_m[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  constexpr int kLane = D / 32;  // elements per lane
  float acc[kLane], sum = 0.f;
#pragma unroll
  for (int e = 0; e < kLane; ++e) acc[e] = 0.f;
  for (int j0 = warp; j0 < np; j0 += 4 * 8) {  // eight pieces' loads in flight
    float2 v[8];
    float x[8][kLane];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t a = at(min(j0 + 4 * i, np - 1));
      v[i] = __ldcg(ml + a);
#pragma unroll
      for (int e = 0; e < kLane; ++e) x[i][e] = __ldcg(p.ws_o + a * D + lane + 32 * e);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float w = v[i].x == top ? 1.f : fast_exp2(v[i].x - top);
      if (j0 + 4 * i >= np) w = 0.f;
      sum += w * v[i].y;
#pragma unroll
      for (int e = 0; e < kLane; ++e) acc[e] += w * x[i][e];
    }
  }
#pragma unroll
  for (int e = 0; e < kLane; ++e) s_o[warp][lane + 32 * e] = acc[e];
  if (lane == 0) s_l[warp] = sum;
  __syncthreads();
  const Rows<T> rows{static_cast<T*>(p.out) + (kChunk ? 0 : b * p.out_stride) +
                         static_cast<int64_t>(hv / p.passes) * p.group * D,
                     p.out_stride, p.group, hv % p.passes * p.per_pass, kChunk};
  T* dst = rows.at(row, D);
  const float inv = 1.f / ((s_l[0] + s_l[1]) + (s_l[2] + s_l[3]));
  for (int d = threadIdx.x; d < D; d += 128)
    dst[d] = from_f32<T>(((s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d])) * inv);
}

// NT: tiles of eight query rows per pass. kChunk: the rows are several tokens of one request.
template <typename T, int D, int S, int NT, bool kChunk>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const Params p) {
  using C = Cfg<D>;
  constexpr int NS = C::kStages;
  constexpr int NP = kUnit / S;  // pages per unit
  constexpr int kRows = S * D / 128;  // 128-byte rows per page tile
  constexpr int kPad = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kWarps * NS * C::kStage);
  float4* s_scale = reinterpret_cast<float4*>(bars + kWarps * NS);  // (sk0, sk1, sv0, sv1)
  int* s_uoff = reinterpret_cast<int*>(s_scale + kWarps * NS);  // first unit of each request
  int* s_ctx = s_uoff + p.batch + 1;

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
    auto units = [&](int i) { return (s_ctx[i] + kUnit - 1) / kUnit; };
    int local = 0;
    for (int i = beg; i < end; ++i) {
      s_ctx[i] = clamp_ctx(kChunk ? (p.causal ? min(p.kv_len, p.q_start + p.q_len) : p.kv_len)
                                  : __ldg(p.ctx_lens + i), max_tokens);
      local += units(i);
    }
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
  const Split split{total, active_warps(total, NW)};  // a segment's pieces are the warps that overlap it
  const bool active = gw < split.warps;
  const int64_t lo = active ? split.first(gw) : 0;
  const int64_t hi = active ? split.first(gw + 1) : 0;

  // (request, head pass, unit) of a stream position; positions fit 32 bits (fast_shape)
  auto locate = [&](int64_t pos64, int& b, int& hv, int& u) {
    const int pos = static_cast<int>(pos64);
    int l = 0, r = B - 1;
    while (l < r) {
      const int mid = (l + r + 1) >> 1;
      if (s_uoff[mid] * HV <= pos) l = mid; else r = mid - 1;
    }
    b = l;
    const int n = s_uoff[l + 1] - s_uoff[l];
    const int rem = pos - s_uoff[l] * HV;
    hv = rem / n;
    u = rem - hv * n;
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
    const int n_pages = (s_ctx[b] + S - 1) / S;
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
      const int n = p.hkv * p.group * D;
      for (int t = 0; t < (kChunk ? p.q_len : 1); ++t)
        for (int i = lane; i < n; i += 32) dst[t * p.out_stride + i] = from_f32<T>(0.f);
    }
  }
  if (!active) return;

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

  // the scales of the unit just issued, beside its stage
  auto put_scales = [&](int64_t pos, int stage) {
    if (lane == static_cast<int>(pos - pbase)) my_scale[stage] = sc_cur;
  };

  // the first loads go out before anything waits for the scales
  int64_t issued = lo;
  for (int s = 0; s < NS && issued < hi; ++s, ++issued) issue(issued, s);
  sc_cur = load_scales(id_cur);
  sc_nxt = load_scales(id_nxt);
  for (int s = 0; s < issued - lo; ++s) put_scales(lo + s, s);
  __syncwarp();  // one lane each wrote them, every lane reads them

  const int gid = lane >> 2;
  const int tig = lane & 3;
  // K: matrix lane / 8, row lane % 8: rows 0-7 / 8-15, bytes 0-15 / 16-31 of each 32
  const int k_tok = row_token((lane & 7) + 8 * ((lane >> 3) & 1));
  const uint32_t k_sw = sw(static_cast<uint32_t>(k_tok * D + 16 * (lane >> 4)));
  // V: row i = 4 t + j of a matrix is k slot 2 t + j (j < 2) or 8 + 2 t + j - 2
  const int vi = lane & 15;
  const int v_tok = row_token(2 * (vi >> 2) + (vi & 1) + 8 * ((vi >> 1) & 1));
  const uint32_t v_sw = sw(static_cast<uint32_t>((16 * (lane >> 4) + v_tok) * D));
  const int r0_tok = gid, r1_tok = 8 + (gid ^ 4);  // tokens of accumulator rows gid, gid + 8

  // The rows of (request b, head pass hv) in a tensor of queries or outputs.
  auto rows_of = [&](auto* base, int64_t stride, int b, int hv) {
    using E = typename std::remove_pointer<decltype(base)>::type;
    const int h = hv / p.passes;
    return Rows<E>{base + (kChunk ? 0 : b * stride) + static_cast<int64_t>(h) * p.group * D, stride, p.group,
                   (hv - h * p.passes) * p.per_pass, kChunk};
  };
  auto count_of = [&](int hv) { return min(p.per_pass, p.rows - hv % p.passes * p.per_pass); };

  uint32_t qf[NT][C::kKK][2];
  float f[NT][2];  // 2^-k scale log2(e) of rows 2 tig and 2 tig + 1
  int lim[NT][2];  // keys that those rows see (kChunk)
  int lim_min = 0;  // ... and the pass's first row, the fewest
  // Query rows in f16; rows beyond the pass are zero.
  auto load_q = [&](int b, int hv) {
    const auto rows = rows_of(static_cast<const T*>(p.q), p.q_stride, b, hv);
    const int n = count_of(hv);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 8 * nt + gid;
      const T* row = rows.at(min(r, n - 1), D) + 4 * tig;
      uint2 w[C::kKK];
      float amax = 0.f;
#pragma unroll
      for (int kk = 0; kk < C::kKK; ++kk) {
        w[kk] = make_uint2(0u, 0u);
        if (r < n) w[kk] = __ldg(reinterpret_cast<const uint2*>(row + 16 * kk));
        const T* e = reinterpret_cast<const T*>(&w[kk]);
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(to_f32(e[i])));
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
        const T* x = reinterpret_cast<const T*>(&w[kk]);
        qf[nt][kk][0] = MmaOp<__half>::pack(to_f32(x[0]) * up, to_f32(x[1]) * up);
        qf[nt][kk][1] = MmaOp<__half>::pack(to_f32(x[2]) * up, to_f32(x[3]) * up);
      }
      f[nt][0] = __shfl_sync(kFull, down, 8 * tig) * p.scale_log2;
      f[nt][1] = __shfl_sync(kFull, down, 8 * tig + 4) * p.scale_log2;
      if constexpr (kChunk) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = (rows.first + min(8 * nt + 2 * tig + i, n - 1)) / p.group;
          lim[nt][i] = p.causal ? min(p.kv_len, p.q_start + t + 1) : p.kv_len;
        }
        lim_min = p.causal ? min(p.kv_len, p.q_start + rows.first / p.group + 1) : p.kv_len;
      }
    }
  };

  uint64_t o[NT][C::kDT][2];  // (d gid | gid + 8) x (rows 2 tig, 2 tig + 1)
  float m[NT][2], l[NT][2];
  int cb, chv, cu;
  locate(lo, cb, chv, cu);
  int cn = s_uoff[cb + 1] - s_uoff[cb];
  int cctx = s_ctx[cb];
  int64_t piece_start = lo;
  bool fresh = true, failed = false;
  int64_t pos = lo;
  int k = 0;

  auto finalize = [&](int64_t piece_end) {
    const auto rows = rows_of(static_cast<T*>(p.out), p.out_stride, cb, chv);
    const int n = count_of(chv);
    const int64_t seg_start = static_cast<int64_t>(s_uoff[cb]) * HV + static_cast<int64_t>(chv) * cn;
    const int64_t seg_end = seg_start + cn;
    const bool whole = piece_start == seg_start && piece_end == seg_end;
    const int64_t slot = static_cast<int64_t>(gw) * 2 + (piece_start == lo ? 0 : 1);
    float* wo = p.ws_o + slot * kPad * D;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float t[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        t[i] = l[nt][i];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) t[i] += __shfl_xor_sync(kFull, t[i], x);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int g = 8 * nt + 2 * tig + i;
        if (g >= n) continue;
        const float inv = 1.f / t[i];
        T* dst = whole ? rows.at(g, D) : nullptr;
#pragma unroll
        for (int dt = 0; dt < C::kDT; ++dt) {
          const int d = 16 * dt + gid;
          float a[2], b[2];
          unpack2(o[nt][dt][0], a[0], a[1]);
          unpack2(o[nt][dt][1], b[0], b[1]);
          if (whole) {
            dst[d] = from_f32<T>(a[i] * inv);
            dst[d + 8] = from_f32<T>(b[i] * inv);
          } else {
            wo[g * D + d] = a[i];
            wo[g * D + d + 8] = b[i];
          }
        }
        if (!whole && gid == 0)
          reinterpret_cast<float2*>(p.ws_ml)[slot * kPad + g] = make_float2(m[nt][i], t[i]);
      }
    }
    if (whole || p.merge_later) return;
    __threadfence();
    __syncwarp();
    int* cnt = p.ws_cnt + cb * HV + chv;
    int old = 0;
    if (lane == 0) old = atomicAdd(cnt, 1);
    old = __shfl_sync(kFull, old, 0);
    const int wa = split.owner(seg_start);
    const int npieces = split.owner(seg_end - 1) - wa + 1;
    if (old != npieces - 1) return;
    __threadfence();
    const int role_a = split.first(wa) == seg_start ? 0 : 1;
    merge_pieces<T, D, kPad>(rows, p.ws_ml, p.ws_o, wa, npieces, role_a, n, lane);
    if (lane == 0) *cnt = 0;
  };

  while (pos < hi) {
    if (fresh) {
      load_q(cb, chv);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int dt = 0; dt < C::kDT; ++dt) o[nt][dt][0] = o[nt][dt][1] = 0ull;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
      piece_start = pos;
      fresh = false;
    }
    const int stage = k % NS;
    if (!__all_sync(kFull, mbar_wait_bounded(bar0 + 8 * stage, static_cast<uint32_t>((k / NS) & 1)))) {
      if (lane == 0) record_error(p.err, PI_ERR_TIMEOUT);
      failed = true;
      break;
    }
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

    // S^T in base-2 units. A warp has a scheduler to itself but for one other, so its own loads
    // and MMAs have to overlap: all of K's fragments are fetched before the first is used, the
    // MMAs run in four chains, and V's fragments are fetched under the softmax.
    constexpr int kHalf = D == 256 ? 4 : C::kKK;  // k steps fetched at once
    float c[NT][2][2][4];
    const uint32_t kbase = ktile + k_sw;
#pragma unroll
    for (int k0 = 0; k0 < C::kKK; k0 += kHalf) {
      uint32_t x[2][kHalf / 2][4];
#pragma unroll
      for (int kk = 0; kk < kHalf; kk += 2)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
          ldmatrix_x4((kbase ^ sw(16 * (k0 + kk))) + 16 * mt * D, x[mt][kk / 2][0], x[mt][kk / 2][1],
                      x[mt][kk / 2][2], x[mt][kk / 2][3]);
#pragma unroll
      for (int kk = 0; kk < kHalf; ++kk)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t a0, a1, a2, a3;
          widen(x[mt][kk / 2][2 * (kk & 1)], a0, a2);
          widen(x[mt][kk / 2][2 * (kk & 1) + 1], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (k0 + kk < 2) mma_f16_zero(c[nt][mt][kk & 1], a0, a1, a2, a3, qf[nt][k0 + kk][0], qf[nt][k0 + kk][1]);
            else mma_f16(c[nt][mt][kk & 1], a0, a1, a2, a3, qf[nt][k0 + kk][0], qf[nt][k0 + kk][1]);
          }
        }
    }
    constexpr int kAhead = D == 256 || NT > 1 ? 4 : C::kDT;  // V tiles fetched at once
    const uint32_t vbase = vtile + v_sw;
    uint32_t y[kAhead][4];
#pragma unroll
    for (int dt = 0; dt < kAhead; ++dt)
      ldmatrix_b8_trans_x2(vbase ^ sw(16 * dt), y[dt][0], y[dt][1], y[dt][2], y[dt][3]);
    // P relative to the unit's maximum (times 256) and to its larger V scale
    float sv = scales.z, w0 = 1.f, w1 = 1.f;
    if (NP == 2) {
      sv = fmaxf(scales.z, scales.w);
      const float ratio = sv > 0.f ? __fdividef(fminf(scales.z, scales.w), sv) : 0.f;
      w0 = scales.z == sv ? 1.f : ratio;
      w1 = scales.w == sv ? 1.f : ratio;
    }
    uint32_t pb[NT][2][2];
    uint64_t al[NT], bs[NT];
    const bool cut = valid < kUnit || (kChunk && (cu + 1) * kUnit > lim_min);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float s[2][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float sk = (NP == 2 && mt == 1) ? scales.y : scales.x;
        const float a = f[nt][0] * sk, b = f[nt][1] * sk;
        s[mt][0] = (c[nt][mt][0][0] + c[nt][mt][1][0]) * a;
        s[mt][1] = (c[nt][mt][0][1] + c[nt][mt][1][1]) * b;
        s[mt][2] = (c[nt][mt][0][2] + c[nt][mt][1][2]) * a;
        s[mt][3] = (c[nt][mt][0][3] + c[nt][mt][1][3]) * b;
      }
      if (cut) {
        const int va = kChunk ? lim[nt][0] - cu * kUnit : valid, vb = kChunk ? lim[nt][1] - cu * kUnit : valid;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          if (16 * mt + r0_tok >= va) s[mt][0] = -INFINITY;
          if (16 * mt + r0_tok >= vb) s[mt][1] = -INFINITY;
          if (16 * mt + r1_tok >= va) s[mt][2] = -INFINITY;
          if (16 * mt + r1_tok >= vb) s[mt][3] = -INFINITY;
        }
      }
      float al2[2], be[2], off[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float u = fmaxf(fmaxf(s[0][i], s[0][i + 2]), fmaxf(s[1][i], s[1][i + 2]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) u = fmaxf(u, __shfl_xor_sync(kFull, u, x));
        const float n = fmaxf(m[nt][i], u);
        // a row that sees nothing of the unit, or of any unit so far: differences to a finite value
        const float n_ref = kChunk && n == -INFINITY ? 0.f : n;
        al2[i] = fast_exp2(m[nt][i] - n_ref);
        be[i] = fast_exp2(u - n_ref);
        off[i] = (kChunk && u == -INFINITY ? 0.f : u) - 8.f;
        m[nt][i] = n;
      }
      float q0 = 0.f, q1 = 0.f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        float e0 = fast_exp2(s[mt][0] - off[0]), e1 = fast_exp2(s[mt][1] - off[1]);
        float e2 = fast_exp2(s[mt][2] - off[0]), e3 = fast_exp2(s[mt][3] - off[1]);
        q0 += e0 + e2;
        q1 += e1 + e3;
        if (NP == 2) {
          const float w = mt ? w1 : w0;
          e0 *= w;
          e1 *= w;
          e2 *= w;
          e3 *= w;
        }
        pb[nt][mt][0] = movmatrix_trans(MmaOp<__half>::pack(e0, e1));
        pb[nt][mt][1] = movmatrix_trans(MmaOp<__half>::pack(e2, e3));
      }
      l[nt][0] = l[nt][0] * al2[0] + be[0] * q0;
      l[nt][1] = l[nt][1] * al2[1] + be[1] * q1;
      al[nt] = pack2(al2[0], al2[1]);
      bs[nt] = pack2(be[0] * sv, be[1] * sv);
    }
#pragma unroll
    for (int d0 = 0; d0 < C::kDT; d0 += kAhead) {
      if (d0 > 0) {
#pragma unroll
        for (int dt = 0; dt < kAhead; ++dt)
          ldmatrix_b8_trans_x2(vbase ^ sw(16 * (d0 + dt)), y[dt][0], y[dt][1], y[dt][2], y[dt][3]);
      }
      float r[NT][kAhead][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int dt = 0; dt < kAhead; ++dt) {
          uint32_t a0, a1, a2, a3;
          widen(y[dt][2 * mt], a0, a2);
          widen(y[dt][2 * mt + 1], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (mt == 0) mma_f16_zero(r[nt][dt], a0, a1, a2, a3, pb[nt][0][0], pb[nt][0][1]);
            else mma_f16(r[nt][dt], a0, a1, a2, a3, pb[nt][1][0], pb[nt][1][1]);
          }
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int dt = 0; dt < kAhead; ++dt) {
          uint64_t* od = o[nt][d0 + dt];
          od[0] = fma2(pack2(r[nt][dt][0], r[nt][dt][1]), bs[nt], mul2(od[0], al[nt]));
          od[1] = fma2(pack2(r[nt][dt][2], r[nt][dt][3]), bs[nt], mul2(od[1], al[nt]));
        }
    }
    __syncwarp();
    if (issued < hi) {
      issue(issued, stage);
      put_scales(issued, stage);
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
        cctx = s_ctx[cb];
        fresh = true;
      }
    } else if (pos == hi) {
      finalize(pos);
    }
  }
  if (failed) {  // loads in flight land before the shared memory is released
    for (int64_t j = k; j < issued - lo; ++j)
      mbar_wait_bounded(bar0 + 8 * static_cast<int>(j % NS), static_cast<uint32_t>((j / NS) & 1));
    if (lane == 0 && !p.merge_later) give_up(split, s_uoff, B, HV, gw, pos, p.ws_cnt);
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
    const int asked = p.ctx_lens != nullptr ? __ldg(p.ctx_lens + b)
                                            : (p.causal ? min(p.kv_len, p.q_start + b + 1) : p.kv_len);
    const int ctx = clamp_ctx(asked, most > 0x7fffffff ? 0x7fffffff : static_cast<int>(most));
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
  cuuint64_t dims[2] = {128, rows};
  cuuint64_t strides[1] = {128};
  cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  return attn::encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
}

struct Layout {
  size_t ml_off, o_off, total;
};
inline size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
// [arrival counters | partial (max, sum) | partial O]; the counters have one place for every
// shape, so zeroed once they stay zero between launches. The block is the 16-bit kernels' too, the
// gather's completion counter at its end included: partials there would stop the next gather.
Layout ws_layout(int head_dim, int sms) {
  Layout L;
  const size_t slots = static_cast<size_t>(sms) * kMaxCtasPerSm * kWarps * 2;
  L.ml_off = align256(kAttnCounterBytes);
  L.o_off = L.ml_off + align256(slots * 8 * kMaxTiles * 2 * sizeof(float));
  L.total = L.o_off + align256(slots * 8 * kMaxTiles * static_cast<size_t>(head_dim) * sizeof(float));
  return L;
}

// Whether the tensor-core kernel takes this; `requests` tables of max_pages pages, `rows` query rows
// per KV head in passes of per_pass.
bool fast_shape(int dtype, int requests, int hkv, int64_t passes, int D, int S, int64_t pages, int64_t max_pages) {
  const int64_t segments = requests * hkv * passes;
  return (dtype == PI_DTYPE_BF16 || dtype == PI_DTYPE_F16) && (D == 64 || D == 128 || D == 256) &&
         (S == 16 || S == 32) && requests <= kMaxBatch && segments <= kMaxSegments &&
         pages * hkv * (S * D / 128) <= 0x7fffffff && pages * hkv <= 0x7fffffff && pages > 0 &&
         max_pages * S <= 0x7fffffff - kUnit &&
         // units are counted in 32 bits
         segments * ((max_pages * S + kUnit - 1) / kUnit) < 0x70000000;
}

template <typename T, int D, int S, int NT, bool kChunk>
int launch(const Params& p, const void* k_pool, const void* v_pool, cudaStream_t stream) {
  auto kern = decode_q8_kernel<T, D, S, NT, kChunk>;
  static std::atomic<int> configured[64];  // per device: the shared memory limit is set
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
  // two CTAs share an SM while the prefix tables leave room for both
  const int per_sm = D <= 128 && 2 * (smem + 1024) <= 228 * 1024 ? 2 : 1;
  const uint64_t rows = static_cast<uint64_t>(p.num_pages) * p.hkv * (S * D / 128);
  CUtensorMap tk, tv;
  if (!pool_map(&tk, k_pool, rows, S * D / 128) || !pool_map(&tv, v_pool, rows, S * D / 128))
    return PI_ERR_CUDA;
  const int64_t segments = static_cast<int64_t>(p.batch) * p.hkv * p.passes;
  Params q = p;
  q.merge_later = segments <= kMergeSegments ? 1 : 0;
  const int ctas = device_sm_count() * per_sm;
  const int rc = cuda_status(launch_kernel(kern, dim3(ctas), dim3(kThreads), smem, stream, tk, tv, q));
  if (rc != PI_OK || !q.merge_later) return rc;
  return cuda_status(launch_kernel(merge_kernel<T, D, 8 * NT, kChunk>,
                                   dim3(static_cast<unsigned>(segments * p.per_pass)), dim3(128), 0, stream, q, S,
                                   ctas * kWarps));
}

// Places the scratch; PI_OK or why not.
int place(Params& p, int head_dim, void* workspace, size_t bytes) {
  const Layout L = ws_layout(head_dim, device_sm_count());
  if (workspace == nullptr || bytes < L.total) return PI_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return PI_ERR_MISALIGNED;
  char* ws = static_cast<char*>(workspace);
  p.ws_cnt = reinterpret_cast<int*>(ws);
  p.ws_ml = reinterpret_cast<float*>(ws + L.ml_off);
  p.ws_o = reinterpret_cast<float*>(ws + L.o_off);
  return PI_OK;
}

int launch_generic(const Params& p, const void* k_pool, const void* v_pool, int hq, int D, int S, int dtype,
                   cudaStream_t stream) {
  const dim3 grid(hq, p.batch < 65535 ? p.batch : 65535);
  const uint8_t* kp = static_cast<const uint8_t*>(k_pool);
  const uint8_t* vp = static_cast<const uint8_t*>(v_pool);
  switch (dtype) {
    case PI_DTYPE_F32:
      return cuda_status(launch_kernel(decode_q8_generic_kernel<float>, grid, dim3(128), 0, stream, p, kp, vp, D, S));
    case PI_DTYPE_BF16:
      return cuda_status(launch_kernel(decode_q8_generic_kernel<__nv_bfloat16>, grid, dim3(128), 0, stream, p, kp, vp, D, S));
    default:
      return cuda_status(launch_kernel(decode_q8_generic_kernel<__half>, grid, dim3(128), 0, stream, p, kp, vp, D, S));
  }
}

}  // namespace q8
}  // namespace pi

extern "C" size_t pi_paged_decode_attn_q8_workspace_bytes(int head_dim) {
  if (head_dim <= 0) return 0;
  return pi::q8::ws_layout(head_dim, pi::device_sm_count()).total;
}

extern "C" size_t pi_paged_decode_attn_q8_ws_zero_bytes(void) {
  return pi::q8::align256(pi::kAttnCounterBytes);
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
  q8::Params p = {};
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
  p.rows = group;
  p.passes = (group + 7) / 8;
  p.per_pass = (group + p.passes - 1) / p.passes;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = err;
  const bool fast = q8::fast_shape(dtype, batch, num_kv_heads, p.passes, head_dim, page_size, num_pages,
                                   max_pages) &&
                    aligned(k_pool, 16) && aligned(v_pool, 16) && aligned(q, 8) && q_stride % 4 == 0;
  if (fast) {
    const int rc = q8::place(p, head_dim, workspace, workspace_bytes);
    if (rc != PI_OK) return rc;
#define PI_Q8(T, D, S) \
  if (head_dim == D && page_size == S) return q8::launch<T, D, S, 1, false>(p, k_pool, v_pool, stream);
#define PI_Q8_ALL(T) PI_Q8(T, 64, 16) PI_Q8(T, 64, 32) PI_Q8(T, 128, 16) PI_Q8(T, 128, 32) \
                     PI_Q8(T, 256, 16) PI_Q8(T, 256, 32)
    if (dtype == PI_DTYPE_BF16) { PI_Q8_ALL(__nv_bfloat16) } else { PI_Q8_ALL(__half) }
#undef PI_Q8_ALL
#undef PI_Q8
  }
  return q8::launch_generic(p, k_pool, v_pool, num_q_heads, head_dim, page_size, dtype, stream);
}

// ---------------------------------------------------------------------------------
// Widened pages, and attention of one request's query tokens
// ---------------------------------------------------------------------------------
namespace pi {
namespace q8 {

// out[i, h, :, :] = pool[ids[i], h, :, :] * scale[ids[i], h], sixteen elements per thread (or one).
// Bound by HBM (one byte read and two written per element). With `identity`, also writes 0, 1, 2, ...:
// the block table of the widened pages.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    page_dequant_kernel(T* out_k, T* out_v, const uint8_t* pool_k, const uint8_t* pool_v, const float* scale_k,
                        const float* scale_v, const int32_t* ids, int32_t* identity, int64_t n_pages, int hkv,
                        int tile, int64_t num_pages, int* err) {
  pdl_wait();
  pdl_trigger();
  const int64_t per_tile = tile / V;
  const int64_t per_pool = n_pages * hkv * per_tile;
  const int64_t total = per_pool * (out_v != nullptr ? 2 : 1);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  if (identity != nullptr)
    for (int64_t i = first; i < n_pages; i += step) identity[i] = static_cast<int32_t>(i);
  for (int64_t x = first; x < total; x += step) {
    const bool is_v = x >= per_pool;
    const int64_t y = is_v ? x - per_pool : x;
    const int64_t block = y / per_tile;  // page of the list * hkv + head
    const int64_t i = block / hkv;
    const int32_t id = __ldg(ids + i);
    const bool ok = id >= 0 && id < num_pages;
    if (!ok) record_error(err, PI_ERR_PAGE_RANGE);
    const int64_t src_block = ok ? id * static_cast<int64_t>(hkv) + (block - i * hkv) : 0;
    const float s = ok ? (is_v ? scale_v : scale_k)[src_block] : 0.f;
    const uint8_t* src = (is_v ? pool_v : pool_k) + src_block * tile + (y - block * per_tile) * V;
    T* dst = (is_v ? out_v : out_k) + y * V;
    // a finite value that f16 cannot hold becomes its largest
    auto value = [&](float v) {
      v = ok ? v * s : 0.f;
      if (std::is_same<T, __half>::value && fabsf(v) > 65504.f && fabsf(v) < INFINITY) v = copysignf(65504.f, v);
      return v;
    };
    if constexpr (V == 16) {
      const uint4 w = ok ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t in[4] = {w.x, w.y, w.z, w.w};
      alignas(16) T vals[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t lo, hi;
        widen(in[q], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
        vals[4 * q] = from_f32<T>(value(a.x));
        vals[4 * q + 1] = from_f32<T>(value(a.y));
        vals[4 * q + 2] = from_f32<T>(value(b.x));
        vals[4 * q + 3] = from_f32<T>(value(b.y));
      }
#pragma unroll
      for (int q = 0; q < static_cast<int>(sizeof(T)); ++q)
        reinterpret_cast<uint4*>(dst)[q] = reinterpret_cast<const uint4*>(vals)[q];
    } else {
      *dst = from_f32<T>(value(ok ? e4m3_value(*src) : 0.f));
    }
  }
}

template <typename T>
int launch_dequant(void* out_k, void* out_v, const void* pool_k, const void* pool_v, const float* scale_k,
                   const float* scale_v, const int32_t* ids, int32_t* identity, int64_t n_pages, int hkv, int tile,
                   int64_t num_pages, int* err, cudaStream_t stream) {
  const bool wide = tile % 16 == 0 && aligned(out_k, 16) && aligned(out_v, 16) && aligned(pool_k, 16) &&
                    aligned(pool_v, 16);
  const int64_t items = n_pages * hkv * (wide ? tile / 16 : tile) * (out_v != nullptr ? 2 : 1);
  int64_t blocks = (items + 255) / 256;
  const int64_t cap = static_cast<int64_t>(device_sm_count()) * 8;
  if (blocks > cap) blocks = cap;
  auto kern = wide ? page_dequant_kernel<T, 16> : page_dequant_kernel<T, 1>;
  return cuda_status(launch_kernel(kern, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                                   static_cast<T*>(out_k), static_cast<T*>(out_v), static_cast<const uint8_t*>(pool_k),
                                   static_cast<const uint8_t*>(pool_v), scale_k, scale_v, ids, identity, n_pages, hkv,
                                   tile, num_pages, err));
}

// Scratch of the widening path: K pages, V pages, their block table.
struct WideLayout {
  size_t v_off, table_off, total;
};
WideLayout wide_layout(int64_t pages, int hkv, int D, int S) {
  WideLayout w;
  const size_t bytes = align256(static_cast<size_t>(pages) * hkv * S * D * 2);
  w.v_off = bytes;
  w.table_off = 2 * bytes;
  w.total = 2 * bytes + align256(static_cast<size_t>(pages) * 4);
  return w;
}

// Many query rows (above PI_Q8_FEW_ROWS): the pages are widened once into scratch and the tcgen05 prefill
// runs on them. Few: the rows ride in the decode kernel, 16 to a pass over the cache (from L2 after
// the first). Measured after 8000 tokens, 32/8 heads of 128: 64 / 128 / 160 / 256 queries take 66 /
// 123 / 144 / 207 us in passes and 154 / 156 / 154 / 153 us widened; with 4 query heads on one KV
// head 128 / 512 queries after 16000 take 41 / 111 us against 270 / 275.
bool widens(int q_len, int kv_len, int hq, int hkv, int D, int S, int dtype) {
  const int G = hq / hkv;
  return (dtype == PI_DTYPE_BF16 || dtype == PI_DTYPE_F16) && (D == 64 || D == 128) && (S == 16 || S == 32) &&
         (G == 1 || G == 2 || G == 4 || G == 8 || G == 16) && kv_len > 0 &&
         static_cast<int64_t>(q_len) * hq > PI_Q8_FEW_ROWS;
}

template <typename T>
int launch_chunk(const Params& p, const void* k_pool, const void* v_pool, int D, int S, cudaStream_t stream) {
#define PI_CHUNK(DIM, PAGE, NT) \
  if (D == DIM && S == PAGE) return launch<T, DIM, PAGE, NT, true>(p, k_pool, v_pool, stream);
  PI_CHUNK(64, 16, 2) PI_CHUNK(64, 32, 2) PI_CHUNK(128, 16, 2) PI_CHUNK(128, 32, 2)
  PI_CHUNK(256, 16, 1) PI_CHUNK(256, 32, 1)
#undef PI_CHUNK
  return PI_ERR_UNSUPPORTED;
}

}  // namespace q8
}  // namespace pi

extern "C" int pi_page_dequant(void* out, const void* pool, const float* scale, const int32_t* page_ids,
                               int64_t n_pages, int kv_heads, int head_dim, int page_size, int64_t num_pages,
                               int dtype, int* err, cudaStream_t stream) {
  using namespace pi;
  const int eb = elem_bytes_of(dtype);
  if (eb == 0) return PI_ERR_UNSUPPORTED;
  if (n_pages < 0 || kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || num_pages < 0 ||
      static_cast<int64_t>(page_size) * head_dim > 0x7fffffff)
    return PI_ERR_BAD_SHAPE;
  if (n_pages == 0) return PI_OK;
  if (!out || !pool || !scale || !page_ids) return PI_ERR_NULL_POINTER;
  if (!aligned(out, eb) || !aligned(scale, 4) || !aligned(page_ids, 4)) return PI_ERR_MISALIGNED;
  const int tile = page_size * head_dim;
  switch (dtype) {
    case PI_DTYPE_F32:
      return q8::launch_dequant<float>(out, nullptr, pool, nullptr, scale, nullptr, page_ids, nullptr, n_pages, kv_heads, tile, num_pages, err, stream);
    case PI_DTYPE_BF16:
      return q8::launch_dequant<__nv_bfloat16>(out, nullptr, pool, nullptr, scale, nullptr, page_ids, nullptr, n_pages, kv_heads, tile, num_pages, err, stream);
    default:
      return q8::launch_dequant<__half>(out, nullptr, pool, nullptr, scale, nullptr, page_ids, nullptr, n_pages, kv_heads, tile, num_pages, err, stream);
  }
}

extern "C" size_t pi_paged_prefill_attn_q8_workspace_bytes(int q_len, int kv_len, int num_q_heads, int num_kv_heads,
                                                           int head_dim, int page_size, int dtype) {
  using namespace pi;
  if (q_len <= 0 || kv_len < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
      head_dim <= 0 || page_size <= 0)
    return 0;
  size_t n = q8::ws_layout(head_dim, device_sm_count()).total;
  if (q8::widens(q_len, kv_len, num_q_heads, num_kv_heads, head_dim, page_size, dtype)) {
    const size_t w = q8::wide_layout((static_cast<int64_t>(kv_len) + page_size - 1) / page_size, num_kv_heads,
                                     head_dim, page_size).total;
    n += w;
  }
  return n;
}

extern "C" int pi_paged_prefill_attn_q8(void* out, const void* q, const void* k_pool, const void* v_pool,
                                        const float* k_scale, const float* v_scale, const int32_t* block_table,
                                        int64_t table_len, int q_len, int kv_len, int q_start, int causal,
                                        int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                        int64_t num_pages, float scale, int dtype, int64_t q_tok_stride,
                                        int64_t out_tok_stride, void* workspace, size_t workspace_bytes, int* err,
                                        cudaStream_t stream) {
  using namespace pi;
  const int eb = elem_bytes_of(dtype);
  if (eb == 0) return PI_ERR_UNSUPPORTED;
  if (q_len < 0 || kv_len < 0 || q_start < 0 || table_len < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads || head_dim <= 0 || page_size <= 0 || num_pages < 0 ||
      static_cast<int64_t>(q_start) + q_len > 0x7fffffff)
    return PI_ERR_BAD_SHAPE;
  if (static_cast<int64_t>(kv_len) > table_len * page_size) return PI_ERR_BAD_SHAPE;
  const int64_t row = static_cast<int64_t>(num_q_heads) * head_dim;
  if (q_tok_stride < row || out_tok_stride < row || row > 0x7fffffff) return PI_ERR_BAD_SHAPE;
  if (head_dim > q8::kGenericMaxD) return PI_ERR_UNSUPPORTED;
  if (q_len == 0) return PI_OK;
  if (!out || !q || !k_pool || !v_pool || !k_scale || !v_scale || (kv_len > 0 && !block_table))
    return PI_ERR_NULL_POINTER;
  if (!aligned(block_table, 4) || !aligned(k_scale, 4) || !aligned(v_scale, 4) || !aligned(q, eb) ||
      !aligned(out, eb))
    return PI_ERR_MISALIGNED;
  const bool aligned_rows = aligned(q, 16) && q_tok_stride % 8 == 0 && aligned(out, 16) && out_tok_stride % 8 == 0 &&
                            aligned(k_pool, 16) && aligned(v_pool, 16);
  const int64_t seen = causal ? (static_cast<int64_t>(q_start) + q_len < kv_len ? q_start + q_len : kv_len) : kv_len;
  const int64_t pages = (seen + page_size - 1) / page_size;
  const size_t narrow_bytes = q8::ws_layout(head_dim, device_sm_count()).total;
  if (num_pages > 0 && aligned_rows && pages * num_kv_heads * page_size <= 0x7fffffff &&
      q8::widens(q_len, kv_len, num_q_heads, num_kv_heads, head_dim, page_size, dtype)) {
    const q8::WideLayout w = q8::wide_layout(pages, num_kv_heads, head_dim, page_size);
    if (workspace == nullptr || workspace_bytes < narrow_bytes + w.total) return PI_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return PI_ERR_MISALIGNED;
    // behind the scratch whose counters stay zero between calls
    char* ws = static_cast<char*>(workspace) + narrow_bytes;
    int32_t* table = reinterpret_cast<int32_t*>(ws + w.table_off);
    const int rc =
        dtype == PI_DTYPE_BF16
            ? q8::launch_dequant<__nv_bfloat16>(ws, ws + w.v_off, k_pool, v_pool, k_scale, v_scale, block_table, table,
                                                pages, num_kv_heads, page_size * head_dim, num_pages, err, stream)
            : q8::launch_dequant<__half>(ws, ws + w.v_off, k_pool, v_pool, k_scale, v_scale, block_table, table, pages,
                                         num_kv_heads, page_size * head_dim, num_pages, err, stream);
    if (rc != PI_OK) return rc;
    return pi_paged_prefill_attn_tc(out, q, ws, ws + w.v_off, table, pages, q_len, static_cast<int>(seen), q_start,
                                    causal, num_q_heads, num_kv_heads, head_dim, page_size, pages, scale, dtype,
                                    q_tok_stride, out_tok_stride, err, stream);
  }
  q8::Params p = {};
  p.out = out;
  p.q = q;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_table;
  p.q_stride = q_tok_stride;
  p.out_stride = out_tok_stride;
  p.num_pages = num_pages;
  p.max_pages = static_cast<int>(num_pages > 0 ? pages : 0);
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.q_len = q_len;
  p.kv_len = num_pages > 0 ? kv_len : 0;
  p.q_start = q_start;
  p.causal = causal ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = err;
  const int64_t rows = static_cast<int64_t>(q_len) * p.group;
  const int per_pass = head_dim == 256 ? 8 : 16;
  const int64_t passes = (rows + per_pass - 1) / per_pass;
  const bool fast = rows <= 0x7fffffff && q8::fast_shape(dtype, 1, num_kv_heads, passes, head_dim, page_size, num_pages, pages) &&
                    aligned(k_pool, 16) && aligned(v_pool, 16) && aligned(q, 8) && q_tok_stride % 4 == 0;
  if (fast) {
    p.batch = 1;
    p.rows = static_cast<int>(rows);
    p.passes = static_cast<int>(passes);
    p.per_pass = per_pass;
    const int rc = q8::place(p, head_dim, workspace, workspace_bytes);
    if (rc != PI_OK) return rc;
    // A workspace for widened pages is lent for the call, and not zeroed by its lender; rows that are
    // not aligned for the tcgen05 kernel come here all the same.
    if (q8::widens(q_len, kv_len, num_q_heads, num_kv_heads, head_dim, page_size, dtype) &&
        cudaMemsetAsync(workspace, 0, kAttnCounterBytes, stream) != cudaSuccess)
      return PI_ERR_CUDA;
    return dtype == PI_DTYPE_BF16 ? q8::launch_chunk<__nv_bfloat16>(p, k_pool, v_pool, head_dim, page_size, stream)
                                  : q8::launch_chunk<__half>(p, k_pool, v_pool, head_dim, page_size, stream);
  }
  p.batch = q_len;  // one table for every token
  p.bt_stride = 0;
  return q8::launch_generic(p, k_pool, v_pool, num_q_heads, head_dim, page_size, dtype, stream);
}
