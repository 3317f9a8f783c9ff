// Rotary append: QK-norm (optional) and rotary positions of any number of new query and key
// rows, and the write of their K/V rows at their slots, in one launch. Pools of 16 or 32-bit
// elements take the rows as they are; pools of e4m3 values carry one power-of-two scale per
// (page, KV head).
//
// Mathematics, for a token at position pos, with R rotated elements of a head of D:
//   x = row, or row / sqrt(mean(row^2) + eps) * w over the head's D elements
//   theta_j = pos * inv_freq[j], j < R / 2; c, s = rope_scale * (cos, sin)(theta_j)
//   (a, b) = (x[j], x[j + R/2]) or (x[2j], x[2j + 1])  ->  (a c - b s, b c + a s)
// and x[R ..] unchanged. The angle is reduced in fp64: pos * inv_freq in fp32 is off by
// pos * 2^-24 radians, 0.06 at position 10^6, where fp64 leaves 10^-10. Everything else is fp32,
// with one rounding to the output type.
//
// 8-bit pools. A block is one page of one KV head. Tokens of one call with consecutive slots
// inside a page form a run; its rows and the rows already in the page before it (offsets
// below the run's first) share the block's scale 2^e:
//   e = max(e of the kept rows, smallest e with amax(new rows) <= 448 * 2^e),
// and a kept row whose scale grows is rescaled by 2^(e_old - e). A power of two loses nothing
// against amax / 448 (e4m3 is a floating format: the step relative to a value is the same) and
// makes rescaling an exponent shift, exact above e4m3's subnormals; values times scale are
// exact in bf16. A run at offset 0 starts the block anew. Rows behind the run keep their bytes.
// A page takes one run per call: two would have to agree on its scale and its kept rows, and they
// belong to CTAs that cannot wait for one another. Where there is an `err` to tell it by, the CTA of a
// run counts the call's tokens that name its page, and where they are more than the run's, no run of
// that page is written. That reads all slots in every such CTA (L2): 8192 tokens take 80 us so
// and 75 without, 64 take 7.1 and 6.4 in a graph, which is why a call without `err` does not look.
//
// What bounds it: every byte is moved once, so HBM; for a step of 64 tokens, latency. A CTA
// takes a tile of tokens and a group of heads, and computes the tile's cosines and sines once
// into shared memory: they serve every head of the group. A lane holds 16 elements of a row,
// eight pairs, so a pair never crosses lanes: two 16-byte loads (16-bit types) eight pairs
// apart in the half layout, adjacent in the interleaved one.
//
// Measured on B200 (32 query and 8 KV heads of 128, bf16, QK-norm): 8192 tokens in 53 us, 3.8 TB/s,
// 0.57 of the measured copy rate; into e4m3 pools 75 us, 0.37. The counters name no single limit: an
// instruction issues in 67 % of the cycles (60 % into e4m3 pools, where 79 registers leave fewer warps),
// waits on loads and on shared memory make up most of the rest, DRAM is at 36 % (23 %). Two rows' loads
// in flight per lane were slower (72 us: 80 registers instead of 56 leave fewer warps). 64 tokens
// take 4.4 and 6.4 us in a graph, the former as decode_prologue.cu does.
#include <type_traits>

#include <cuda_fp8.h>

#include "pi_common.cuh"

namespace pi {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxTile = 8;    // tokens per CTA (16: 59 us against 54 for 8192 tokens)
constexpr int kMinExp = -118;  // smallest scale exponent: 2^e and 2^-e are normal floats

struct AppendParams {
  void* q_out;
  char* k_pool;
  char* v_pool;
  float* k_scale;  // [num_pages, hkv], 8-bit pools only
  float* v_scale;
  const void* q_in;
  const void* k_in;
  const void* v_in;
  const void* q_norm_w;
  const void* k_norm_w;
  const float* inv_freq;        // [pairs]
  const int64_t* positions;     // [n]
  const int64_t* slot_mapping;  // [n]
  int64_t q_out_stride, q_in_stride, k_in_stride, v_in_stride;
  int64_t n_tokens, num_slots;
  float eps, rope_scale;
  int hq, hkv, head_dim, page_size, pairs, interleaved, tile, groups;
  int* err;
};

// cos and sin of pos * inv_freq, times rope_scale. In turns the reduction is a subtraction
// of the nearest whole number, exact in fp64; what rounding to fp32 takes off the reduced
// angle is put back to first order.
__device__ __forceinline__ float2 cos_sin(int64_t pos, float inv_freq, float rope_scale) {
  constexpr double kInvPi = 0.31830988618379067154;
  double half_turns = static_cast<double>(pos) * static_cast<double>(inv_freq) * kInvPi;
  half_turns -= 2.0 * rint(0.5 * half_turns);
  const float x = static_cast<float>(half_turns);
  const float rest = static_cast<float>(half_turns - static_cast<double>(x)) * 3.14159265f;
  float s, c;
  sincospif(x, &s, &c);
  return make_float2((c - rest * s) * rope_scale, (s + rest * c) * rope_scale);
}

// ---- 16 elements of a row: lane l of the row's D / 16 holds elements [d_a, d_a + 8) and
// [d_b, d_b + 8); x[0..7] and x[8..15]. ------------------------------------------------

struct LaneCols {
  int a, b;
  int pair;      // first of the lane's eight pairs, or -1: not rotated
};

__device__ __forceinline__ LaneCols lane_cols(int l, int pairs, bool interleaved) {
  const int rotated = pairs / 8;  // lanes that rotate
  if (l >= rotated) return {16 * l, 16 * l + 8, -1};
  if (interleaved) return {16 * l, 16 * l + 8, 8 * l};
  return {8 * l, 8 * l + pairs, 8 * l};
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 u = __ldg(reinterpret_cast<const float4*>(p));
    const float4 v = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  } else {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* h = reinterpret_cast<const T*>(&w[i]);
      x[2 * i] = to_f32(h[0]);
      x[2 * i + 1] = to_f32(h[1]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(MmaOp<T>::pack(x[0], x[1]), MmaOp<T>::pack(x[2], x[3]),
                                              MmaOp<T>::pack(x[4], x[5]), MmaOp<T>::pack(x[6], x[7]));
  }
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ void store8_e4m3(uint8_t* p, const float* x, float inv) {
  *reinterpret_cast<uint2*>(p) =
      make_uint2(e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                 e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv));
}

// Division by the root mean square of a row. x * rinv is a rounding off the quotient twice over; with
// its residual x - y rms put back (one Newton step on the quotient) it is the quotient rounded once in
// all but rare cases, which keeps a value next to an e4m3 border on its side. A root that overflowed
// (an infinity in the row, or a sum of squares past fp32) has no residual, inf * 0: it is taken as 0
// there, so that x / inf = 0 for every finite x and NaN for an infinity, as the division gives. (Chosen
// in the root, not per element: a select for each took eight more registers and 5 % of the time.)
struct RowNorm {
  float rms, rinv;
};

__device__ __forceinline__ RowNorm row_norm(float mean_square, float eps) {
  const float rms = sqrtf(mean_square + eps);
  return {rms < INFINITY ? rms : 0.f, 1.f / rms};
}

__device__ __forceinline__ float quotient(float x, const RowNorm& n) {
  const float y = x * n.rinv;
  return fmaf(fmaf(-y, n.rms, x), n.rinv, y);
}

// Norm (over the row's L lanes; every lane of the warp calls) and rotation in place.
template <typename Ti, int L>
__device__ __forceinline__ void norm_rotate(float (&x)[16], const LaneCols& c, const Ti* w,
                                            float eps, const float2* table, bool interleaved) {
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const RowNorm n = row_norm(ss / static_cast<float>(16 * L), eps);
    float wv[16];
    load8(w + c.a, wv);
    load8(w + c.b, wv + 8);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = quotient(x[i], n) * wv[i];
  }
  if (c.pair < 0) return;
  const float4* t = reinterpret_cast<const float4*>(table + c.pair);  // two (cos, sin) pairs each
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float4 cs = t[i / 2];
    if (interleaved) {
      const float a0 = x[2 * i], b0 = x[2 * i + 1], a1 = x[2 * i + 2], b1 = x[2 * i + 3];
      x[2 * i] = a0 * cs.x - b0 * cs.y;
      x[2 * i + 1] = b0 * cs.x + a0 * cs.y;
      x[2 * i + 2] = a1 * cs.z - b1 * cs.w;
      x[2 * i + 3] = b1 * cs.z + a1 * cs.w;
    } else {
      const float a0 = x[i], b0 = x[i + 8], a1 = x[i + 1], b1 = x[i + 9];
      x[i] = a0 * cs.x - b0 * cs.y;
      x[i + 8] = b0 * cs.x + a0 * cs.y;
      x[i + 1] = a1 * cs.z - b1 * cs.w;
      x[i + 9] = b1 * cs.z + a1 * cs.w;
    }
  }
}

// |x| where it is finite, else 0: what a block's scale goes by.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// Smallest e >= kMinExp with amax <= 448 * 2^e; 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kMinExp);
}

// Smallest e >= kMinExp with s <= 2^e for a scale that a block already has.
__device__ __forceinline__ int kept_exp(float s) {
  if (!(s > 0.f && s < INFINITY)) return kMinExp;
  const uint32_t u = __float_as_uint(s);
  return max(static_cast<int>(u >> 23) - 127 + ((u & 0x7fffffu) != 0 ? 1 : 0), kMinExp);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Four e4m3 values times ratio, rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t v, float ratio) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v >> (16 * i)), __NV_E4M3);
    const float2 g = __half22float2(__half2(h));
    f[2 * i] = g.x * ratio;
    f[2 * i + 1] = g.y * ratio;
  }
  return e4m3x4(f[0], f[1], f[2], f[3]);
}

// The runs of a tile: token t starts one if it has a slot and does not continue its
// predecessor's page; the run goes on while the slots count up inside the page.
__device__ __forceinline__ bool run_starts(const int64_t* slots, int i, int page_size) {
  // slots[i] is the slot of the token before token i of the tile
  const int64_t s = slots[i + 1];
  return s >= 0 && !(slots[i] >= 0 && s == slots[i] + 1 && s % page_size != 0);
}

// Adds to named[i], for each token i of the tile that starts a run (a bit of `starts`), the call's tokens
// whose page has the same low 32 bits. All threads call.
template <int S>
__device__ __noinline__ void count_named(const int64_t* slot_mapping, int64_t n, uint32_t starts, const int64_t* slots,
                                         int* named, int tid) {
  constexpr int kShift = S == 16 ? 4 : 5;
  static_assert(S == 1 << kShift, "pages of 16 or 32 tokens");
  constexpr int kBatch = 16;  // loads in flight
  auto count = [&](const uint32_t* page, int batch) {
    for (uint32_t left = starts; left != 0; left &= left - 1) {
      const int i = __ffs(left) - 1;
      const uint32_t own = static_cast<uint32_t>(slots[i + 1] >> kShift);
      int c = 0;
#pragma unroll
      for (int e = 0; e < batch; ++e) c += page[e] == own ? 1 : 0;
      if (c != 0) atomicAdd(named + i, c);
    }
  };
  int64_t j = tid;
  for (; j + (kBatch - 1) * kThreads < n; j += kBatch * kThreads) {
    uint32_t page[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e)
      page[e] = static_cast<uint32_t>(__ldg(slot_mapping + j + e * kThreads) >> kShift);
    count(page, kBatch);
  }
  for (; j < n; j += kThreads) {
    const uint32_t page = static_cast<uint32_t>(__ldg(slot_mapping + j) >> kShift);
    count(&page, 1);
  }
}

// kPoolBits 8: K and V rows go to e4m3 blocks (To is then q's output type); else To is the
// pools' type too. S: page size (8-bit pools only).
template <typename Ti, typename To, int D, bool k8, int S>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const AppendParams p) {
  pdl_wait();  // the rows are the previous kernel's output
  pdl_trigger();
  constexpr int L = D / 16;  // lanes per row
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tile;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.tile), p.n_tokens - t0));
  // 8-bit: the tile's runs may reach S - 1 tokens past it
  const int ext = k8 ? static_cast<int>(min(static_cast<int64_t>(p.tile + S - 1), p.n_tokens - t0)) : nt;
  const int pairs = p.pairs;
  const bool il = p.interleaved != 0;
  float2* table = reinterpret_cast<float2*>(smem);  // [tile (+ S - 1)][pairs]
  const int g = blockIdx.y, ng = p.groups;
  // group i's first head: n / ng heads each, one more for the first n % ng (n * i may pass 32 bits)
  auto first = [&](int n, int i) { return n / ng * i + min(i, n % ng); };
  const int q0 = first(p.hq, g), q1 = first(p.hq, g + 1);
  const int h0 = first(p.hkv, g), h1 = first(p.hkv, g + 1);
  __shared__ int64_t s_slot[k8 ? 64 + 32 : 1];
  __shared__ float s_max[2][kThreads / 32];
  __shared__ int s_named[kMaxTile];  // 8-bit: tokens of the call that name the page of the run at a token
  // Where a token's K and V rows go (elements from the pools' start, head 0), -1: nowhere. Worked out
  // once per token: the 64-bit division per row cost more than moving it.
  __shared__ int64_t s_dst[k8 ? 1 : kMaxTile];
  if constexpr (!k8) {
    if (tid < nt) {
      const int64_t slot = __ldg(p.slot_mapping + t0 + tid);
      const int64_t page = slot / p.page_size;
      if (slot >= p.num_slots && g == 0) record_error(p.err, PI_ERR_SLOT_RANGE);
      s_dst[tid] = slot < 0 || slot >= p.num_slots
                       ? -1 : (page * p.hkv * p.page_size + (slot - page * p.page_size)) * D;
    }
  }
  int covered = nt;  // tokens whose rows this CTA touches
  if constexpr (k8) {
    for (int i = tid; i <= ext; i += kThreads)
      s_slot[i] = t0 + i == 0 ? -1 : __ldg(p.slot_mapping + t0 + i - 1);
    if (tid < kMaxTile) s_named[tid] = 0;
    __syncthreads();
    // the last run may go on behind the tile
    if (h1 > h0 && s_slot[nt] >= 0)
      while (covered < ext && s_slot[covered + 1] == s_slot[covered] + 1 && s_slot[covered + 1] % S != 0)
        ++covered;
    if (p.err != nullptr && h1 > h0) {
      uint32_t starts = 0;
      for (int i = 0; i < nt; ++i) starts |= run_starts(s_slot, i, S) ? 1u << i : 0u;
      if (starts != 0) count_named<S>(p.slot_mapping, p.n_tokens, starts, s_slot, s_named, tid);
    }
  }
  for (int i = tid; i < covered * pairs; i += kThreads) {
    const int t = i / pairs;
    table[i] = cos_sin(__ldg(p.positions + t0 + t), __ldg(p.inv_freq + i - t * pairs), p.rope_scale);
  }
  __syncthreads();

  const int l = tid % L;
  const LaneCols cols = lane_cols(l, pairs, il);
  // q rows, and without 8-bit blocks the K and V rows too: one row per L lanes
  const int nq = q1 - q0;
  const int rows = nq + (k8 ? 0 : 2 * (h1 - h0));
  const int total = nt * rows;
  constexpr int kStep = kThreads / L;
  for (int base = 0; base < total; base += kStep) {
    const int r = base + tid / L;
    const bool live = r < total;
    const int t = live ? r / rows : 0;
    const int i = live ? r - t * rows : 0;
    const int kind = i < nq ? 0 : (i < nq + (h1 - h0) ? 1 : 2);
    const int64_t tok = t0 + t;
    const Ti* src;
    To* dst;
    bool write = live;
    if (kind == 0) {
      src = static_cast<const Ti*>(p.q_in) + tok * p.q_in_stride + (q0 + i) * D;
      dst = static_cast<To*>(p.q_out) + tok * p.q_out_stride + (q0 + i) * D;
    } else {
      const int h = h0 + i - nq - (kind == 2 ? h1 - h0 : 0);
      src = kind == 1 ? static_cast<const Ti*>(p.k_in) + tok * p.k_in_stride + h * D
                      : static_cast<const Ti*>(p.v_in) + tok * p.v_in_stride + h * D;
      const int64_t at = s_dst[k8 ? 0 : t];
      write = live && at >= 0;
      // (64 bits: a page of many tokens and heads may hold more than 2^31 elements)
      dst = reinterpret_cast<To*>(kind == 1 ? p.k_pool : p.v_pool) + at +
            h * (static_cast<int64_t>(p.page_size) * D);
    }
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
    if (live) {
      load8(src + cols.a, x);
      load8(src + cols.b, x + 8);
    }
    // A warp of V rows alone skips the norm and the rotation; in a mixed one every lane takes part
    // in the norm's shuffles, and the V lanes keep their rows.
    if (__any_sync(0xffffffffu, kind != 2)) {
      float y[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = x[e];
      norm_rotate<Ti, L>(y, cols, static_cast<const Ti*>(kind == 0 ? p.q_norm_w : p.k_norm_w), p.eps,
                         table + t * pairs, il);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = kind == 2 ? x[e] : y[e];
    }
    if (write) {
      store8(dst + cols.a, x);
      store8(dst + cols.b, x + 8);
    }
  }
  if constexpr (k8) {
    // Blocks: the CTA's threads hold a run's K and V rows of one head (kPass rows x 16
    // elements each), find both maxima, and write the rows in the block's scale.
    constexpr int kRowsPerPass = kThreads / L;
    constexpr int kPass = (S + kRowsPerPass - 1) / kRowsPerPass;
    for (int i = 0; i < nt; ++i) {
      if (!run_starts(s_slot, i, S)) continue;
      const int64_t slot = s_slot[i + 1];
      if (slot >= p.num_slots) {
        if (tid == 0) record_error(p.err, PI_ERR_SLOT_RANGE);
        continue;
      }
      const int64_t page = slot / S;
      const int off = static_cast<int>(slot - page * S);
      int n = 1;
      while (i + n < covered && off + n < S && s_slot[i + 1 + n] == slot + n) ++n;
      if (p.err != nullptr && h1 > h0 && s_named[i] != n) {
        // other tokens name the page, or slots far outside the pool whose pages are alike in 32 bits
        bool other = false;
        for (int64_t j = tid; j < p.n_tokens; j += kThreads)
          other |= static_cast<uint64_t>(__ldg(p.slot_mapping + j) - (slot - off)) < S &&
                   (j < t0 + i || j >= t0 + i + n);
        if (__syncthreads_or(other)) {
          if (tid == 0) record_error(p.err, PI_ERR_PAGE_SHARED);
          continue;
        }
      }
      for (int h = h0; h < h1; ++h) {
        const int64_t block = page * p.hkv + h;
        float k[kPass][16], v[kPass][16];
        float km = 0.f, vm = 0.f;
#pragma unroll
        for (int ps = 0; ps < kPass; ++ps) {
          const int r = ps * kRowsPerPass + tid / L;
#pragma unroll
          for (int e = 0; e < 16; ++e) k[ps][e] = v[ps][e] = 0.f;
          if (r < n) {
            const int64_t tok = t0 + i + r;
            const Ti* ks = static_cast<const Ti*>(p.k_in) + tok * p.k_in_stride + h * D;
            const Ti* vs = static_cast<const Ti*>(p.v_in) + tok * p.v_in_stride + h * D;
            load8(ks + cols.a, k[ps]);
            load8(ks + cols.b, k[ps] + 8);
            load8(vs + cols.a, v[ps]);
            load8(vs + cols.b, v[ps] + 8);
          }
          norm_rotate<Ti, L>(k[ps], cols, static_cast<const Ti*>(p.k_norm_w), p.eps,
                             table + (i + min(r, n - 1)) * pairs, il);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            km = fmaxf(km, finite_abs(k[ps][e]));
            vm = fmaxf(vm, finite_abs(v[ps][e]));
          }
        }
        const float old_k = off > 0 ? p.k_scale[block] : 0.f;
        const float old_v = off > 0 ? p.v_scale[block] : 0.f;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
          km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, o));
          vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
        }
        if ((tid & 31) == 0) {
          s_max[0][tid >> 5] = km;
          s_max[1][tid >> 5] = vm;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
          km = fmaxf(km, s_max[0][w]);
          vm = fmaxf(vm, s_max[1][w]);
        }
        __syncthreads();  // s_max is written again for the next head; the old scales are read
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const float old = kv ? old_v : old_k;
          int e = scale_exp(kv ? vm : km);
          if (off > 0) e = max(e, kept_exp(old));
          const float s = exp2_int(e);
          uint8_t* tile = reinterpret_cast<uint8_t*>(kv ? p.v_pool : p.k_pool) + block * (S * D);
          if (off > 0 && old != s) {  // the kept rows move to the larger scale
            const float ratio = old / s;
            for (int c = tid; c < off * (D / 16); c += kThreads) {
              uint4 w = reinterpret_cast<uint4*>(tile)[c];
              w.x = rescale4(w.x, ratio);
              w.y = rescale4(w.y, ratio);
              w.z = rescale4(w.z, ratio);
              w.w = rescale4(w.w, ratio);
              reinterpret_cast<uint4*>(tile)[c] = w;
            }
          }
          if (tid == 0 && (off == 0 || old != s)) (kv ? p.v_scale : p.k_scale)[block] = s;
          const float inv = exp2_int(-e);
#pragma unroll
          for (int ps = 0; ps < kPass; ++ps) {
            const int r = ps * kRowsPerPass + tid / L;
            if (r < n) {
              uint8_t* row = tile + (off + r) * D;
              store8_e4m3(row + cols.a, kv ? v[ps] : k[ps], inv);
              store8_e4m3(row + cols.b, kv ? v[ps] + 8 : k[ps] + 8, inv);
            }
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// Any other shape, alignment or page size: one element at a time, one warp per row.
// ---------------------------------------------------------------------------------------

// Element d of the (normed, rotated) row; `norm` is not looked at without weights.
template <typename Ti>
__device__ float rotated_element(const AppendParams& p, const Ti* src, const Ti* w, const RowNorm& norm,
                                 int64_t pos, int d) {
  auto at = [&](int i) {
    const float x = to_f32(src[i]);
    if (w == nullptr) return x;
    return quotient(x, norm) * to_f32(w[i]);
  };
  const int n = p.pairs;
  if (d >= 2 * n) return at(d);
  const int j = p.interleaved ? d / 2 : (d < n ? d : d - n);
  const bool second = p.interleaved ? (d & 1) != 0 : d >= n;
  const int other = p.interleaved ? d ^ 1 : (second ? d - n : d + n);
  const float2 cs = cos_sin(pos, __ldg(p.inv_freq + j), p.rope_scale);
  return second ? at(d) * cs.x + at(other) * cs.y : at(d) * cs.x - at(other) * cs.y;
}

template <typename Ti>
__device__ RowNorm norm_of_row(const AppendParams& p, const Ti* src, const Ti* w, int lane) {
  if (w == nullptr) return {1.f, 1.f};
  float ss = 0.f;
  for (int d = lane; d < p.head_dim; d += 32) {
    const float x = to_f32(src[d]);
    ss += x * x;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return row_norm(ss / static_cast<float>(p.head_dim), p.eps);
}

template <typename Ti, typename To, bool k8>
__global__ void __launch_bounds__(kThreads) rope_append_generic_kernel(const AppendParams p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = kThreads / 32;
  const int D = p.head_dim, S = p.page_size;
  const int rows = p.hq + (k8 ? 0 : 2 * p.hkv);
  const Ti* qw = static_cast<const Ti*>(p.q_norm_w);
  const Ti* kw = static_cast<const Ti*>(p.k_norm_w);
  for (int64_t t = blockIdx.x; t < p.n_tokens; t += gridDim.x) {
    const int64_t pos = __ldg(p.positions + t);
    const int64_t slot = __ldg(p.slot_mapping + t);
    for (int i = warp; i < rows; i += nw) {
      const int kind = i < p.hq ? 0 : (i < p.hq + p.hkv ? 1 : 2);
      if (kind == 0) {
        const Ti* src = static_cast<const Ti*>(p.q_in) + t * p.q_in_stride + static_cast<int64_t>(i) * D;
        To* dst = static_cast<To*>(p.q_out) + t * p.q_out_stride + static_cast<int64_t>(i) * D;
        const RowNorm norm = norm_of_row(p, src, qw, lane);
        for (int d = lane; d < D; d += 32)
          dst[d] = from_f32<To>(rotated_element(p, src, qw, norm, pos, d));
        continue;
      }
      if (slot < 0) continue;
      if (slot >= p.num_slots) {
        if (lane == 0) record_error(p.err, PI_ERR_SLOT_RANGE);
        continue;
      }
      const int h = i - p.hq - (kind == 2 ? p.hkv : 0);
      const int64_t page = slot / S;
      To* dst = reinterpret_cast<To*>(kind == 1 ? p.k_pool : p.v_pool) +
                ((page * p.hkv + h) * S + (slot - page * S)) * D;
      if (kind == 1) {
        const Ti* src = static_cast<const Ti*>(p.k_in) + t * p.k_in_stride + static_cast<int64_t>(h) * D;
        const RowNorm norm = norm_of_row(p, src, kw, lane);
        for (int d = lane; d < D; d += 32)
          dst[d] = from_f32<To>(rotated_element(p, src, kw, norm, pos, d));
      } else {
        const Ti* src = static_cast<const Ti*>(p.v_in) + t * p.v_in_stride + static_cast<int64_t>(h) * D;
        for (int d = lane; d < D; d += 32) dst[d] = from_f32<To>(to_f32(src[d]));
      }
    }
    if constexpr (k8) {
      // the CTA of a run's first token writes the run, a warp per (head, K or V)
      if (slot < 0) continue;
      const int64_t prev = t > 0 ? __ldg(p.slot_mapping + t - 1) : -1;
      if (prev >= 0 && slot == prev + 1 && slot % S != 0) continue;
      if (slot >= p.num_slots) {
        if (threadIdx.x == 0) record_error(p.err, PI_ERR_SLOT_RANGE);
        continue;
      }
      const int64_t page = slot / S;
      const int off = static_cast<int>(slot - page * S);
      int n = 1;
      while (t + n < p.n_tokens && off + n < S && __ldg(p.slot_mapping + t + n) == slot + n) ++n;
      bool other = false;
      for (int64_t j = threadIdx.x; p.err != nullptr && j < p.n_tokens; j += kThreads)
        other |= static_cast<uint64_t>(__ldg(p.slot_mapping + j) - (slot - off)) < static_cast<uint64_t>(S) &&
                 (j < t || j >= t + n);
      if (__syncthreads_or(other)) {
        if (threadIdx.x == 0) record_error(p.err, PI_ERR_PAGE_SHARED);
        continue;
      }
      for (int i = warp; i < 2 * p.hkv; i += nw) {
        const bool is_v = i >= p.hkv;
        const int h = is_v ? i - p.hkv : i;
        const int64_t stride = is_v ? p.v_in_stride : p.k_in_stride;
        const Ti* src = static_cast<const Ti*>(is_v ? p.v_in : p.k_in) + t * stride + static_cast<int64_t>(h) * D;
        const int64_t block = page * p.hkv + h;
        uint8_t* tile = reinterpret_cast<uint8_t*>(is_v ? p.v_pool : p.k_pool) + block * S * D;
        float* scale = (is_v ? p.v_scale : p.k_scale) + block;
        auto norm_at = [&](int r) { return norm_of_row(p, src + r * stride, is_v ? nullptr : kw, lane); };
        auto value = [&](int r, const RowNorm& norm, int d) {
          const Ti* row = src + r * stride;
          return is_v ? to_f32(row[d]) : rotated_element(p, row, kw, norm, __ldg(p.positions + t + r), d);
        };
        float m = 0.f;
        for (int r = 0; r < n; ++r) {
          const RowNorm norm = norm_at(r);
          for (int d = lane; d < D; d += 32) m = fmaxf(m, finite_abs(value(r, norm, d)));
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        int e = scale_exp(m);
        const float old = off > 0 ? *scale : 0.f;
        if (off > 0) e = max(e, kept_exp(old));
        const float s = exp2_int(e);
        __syncwarp();  // every lane has read the old scale
        if (off > 0 && old != s) {
          const float ratio = old / s;
          for (int c = lane; c < off * D; c += 32) tile[c] = static_cast<uint8_t>(rescale4(tile[c], ratio));
        }
        if (lane == 0 && (off == 0 || old != s)) *scale = s;
        const float inv = exp2_int(-e);
        for (int r = 0; r < n; ++r) {
          const RowNorm norm = norm_at(r);
          for (int d = lane; d < D; d += 32)
            tile[(off + r) * D + d] = static_cast<uint8_t>(
                __nv_cvt_float_to_fp8(value(r, norm, d) * inv, __NV_SATFINITE, __NV_E4M3));
        }
      }
    }
  }
}

template <typename Ti, typename To, bool k8>
int launch_generic(const AppendParams& p, cudaStream_t stream) {
  const int64_t cap = static_cast<int64_t>(device_sm_count()) * 16;
  const unsigned grid = static_cast<unsigned>(p.n_tokens < cap ? p.n_tokens : cap);
  return cuda_status(launch_kernel(rope_append_generic_kernel<Ti, To, k8>, dim3(grid), dim3(kThreads), 0,
                                   stream, p));
}

template <typename Ti, typename To, int D, bool k8, int S>
int launch_fast(AppendParams p, cudaStream_t stream) {
  // Few tokens: one per tile and the heads over many CTAs, so that a step's loads run on the
  // whole GPU at once; many: tiles of tokens share their cosines and sines.
  const int64_t n = p.n_tokens;
  const int64_t sms = device_sm_count();
  p.tile = n >= 16 * sms ? kMaxTile : (n >= 4 * sms ? 4 : 1);
  const int64_t tiles = (n + p.tile - 1) / p.tile;
  int groups = 1;
  while (groups < p.hkv && tiles * groups < 8 * sms) groups *= 2;
  p.groups = groups;
  if (tiles > 0x7fffffff) return PI_ERR_BAD_SHAPE;
  const size_t smem = static_cast<size_t>(p.tile + (k8 ? S - 1 : 0)) * p.pairs * sizeof(float2);
  auto kern = rope_append_kernel<Ti, To, D, k8, S>;
  return cuda_status(launch_kernel(kern, dim3(static_cast<unsigned>(tiles), groups), dim3(kThreads), smem,
                                   stream, p));
}

template <typename Ti, typename To, bool k8>
int launch_append(const AppendParams& p, bool fast, cudaStream_t stream) {
  if (!fast) return launch_generic<Ti, To, k8>(p, stream);
#define PI_APPEND(DIM)                                                          \
  if (p.head_dim == DIM) {                                                      \
    if constexpr (k8) {                                                         \
      if (p.page_size == 16) return launch_fast<Ti, To, DIM, true, 16>(p, stream); \
      return launch_fast<Ti, To, DIM, true, 32>(p, stream);                     \
    } else {                                                                    \
      return launch_fast<Ti, To, DIM, false, 0>(p, stream);                     \
    }                                                                           \
  }
  PI_APPEND(64)
  PI_APPEND(128)
  PI_APPEND(256)
#undef PI_APPEND
  return PI_ERR_UNSUPPORTED;
}

template <typename Ti>
int dispatch_pool(const AppendParams& p, int pool_dtype, bool fast, cudaStream_t stream) {
  switch (pool_dtype) {
    case PI_DTYPE_F32: return launch_append<Ti, float, false>(p, fast, stream);
    case PI_DTYPE_BF16: return launch_append<Ti, __nv_bfloat16, false>(p, fast, stream);
    case PI_DTYPE_F16: return launch_append<Ti, __half, false>(p, fast, stream);
    case PI_DTYPE_E4M3: return launch_append<Ti, Ti, true>(p, fast, stream);
    default: return PI_ERR_UNSUPPORTED;
  }
}

}  // namespace
}  // namespace pi

extern "C" int pi_rope_append(void* q_out, int64_t q_out_stride, void* k_pool, void* v_pool,
                              float* k_scale, float* v_scale, const void* q_in, int64_t q_in_stride,
                              const void* k_in, int64_t k_in_stride, const void* v_in,
                              int64_t v_in_stride, int in_dtype, const void* q_norm_w,
                              const void* k_norm_w, float eps, const float* inv_freq, int rot_pairs,
                              int interleaved, float rope_scale, const int64_t* positions,
                              const int64_t* slot_mapping, int64_t n_tokens, int num_q_heads,
                              int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                              int pool_dtype, int* err, cudaStream_t stream) {
  using namespace pi;
  const int in_bytes = elem_bytes_of(in_dtype);
  const bool k8 = pool_dtype == PI_DTYPE_E4M3;
  if (in_bytes == 0 || (!k8 && elem_bytes_of(pool_dtype) == 0)) return PI_ERR_UNSUPPORTED;
  if (n_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || page_size <= 0 ||
      num_pages < 0 || rot_pairs < 0 || 2 * static_cast<int64_t>(rot_pairs) > head_dim)
    return PI_ERR_BAD_SHAPE;
  const int64_t q_row = static_cast<int64_t>(num_q_heads) * head_dim;
  const int64_t kv_row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (q_row > 0x7fffffff || kv_row > 0x7fffffff ||
      static_cast<int64_t>(page_size) * head_dim > 0x7fffffff)
    return PI_ERR_BAD_SHAPE;
  if (q_out_stride < q_row || q_in_stride < q_row || k_in_stride < kv_row || v_in_stride < kv_row)
    return PI_ERR_BAD_SHAPE;
  if (!(eps >= 0.f)) return PI_ERR_BAD_SHAPE;
  if (n_tokens == 0) return PI_OK;
  if (!q_out || !k_pool || !v_pool || !q_in || !k_in || !v_in || !positions || !slot_mapping ||
      (rot_pairs > 0 && !inv_freq) || (k8 && (!k_scale || !v_scale)))
    return PI_ERR_NULL_POINTER;
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr)) return PI_ERR_NULL_POINTER;
  if (!aligned(positions, 8) || !aligned(slot_mapping, 8) || !aligned(inv_freq, 4) ||
      !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return PI_ERR_MISALIGNED;
  const int out_bytes = k8 ? in_bytes : elem_bytes_of(pool_dtype);
  if (!aligned(q_in, in_bytes) || !aligned(k_in, in_bytes) || !aligned(v_in, in_bytes) ||
      !aligned(q_norm_w, in_bytes) || !aligned(k_norm_w, in_bytes) || !aligned(q_out, out_bytes) ||
      (!k8 && (!aligned(k_pool, out_bytes) || !aligned(v_pool, out_bytes))))
    return PI_ERR_MISALIGNED;
  AppendParams p;
  p.q_out = q_out;
  p.k_pool = static_cast<char*>(k_pool);
  p.v_pool = static_cast<char*>(v_pool);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.q_in = q_in;
  p.k_in = k_in;
  p.v_in = v_in;
  p.q_norm_w = q_norm_w;
  p.k_norm_w = k_norm_w;
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.slot_mapping = slot_mapping;
  p.q_out_stride = q_out_stride;
  p.q_in_stride = q_in_stride;
  p.k_in_stride = k_in_stride;
  p.v_in_stride = v_in_stride;
  p.n_tokens = n_tokens;
  p.num_slots = num_pages * page_size;
  p.eps = eps;
  p.rope_scale = rope_scale;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.head_dim = head_dim;
  p.page_size = page_size;
  p.pairs = rot_pairs;
  p.interleaved = interleaved ? 1 : 0;
  p.tile = 1;
  p.groups = 1;
  p.err = err;
  // The vector kernel moves whole 16-byte pieces and rotates eight pairs per lane.
  const bool fast =
      (head_dim == 64 || head_dim == 128 || head_dim == 256) && rot_pairs % 8 == 0 &&
      (!k8 || page_size == 16 || page_size == 32) && aligned(q_in, 16) && aligned(k_in, 16) &&
      aligned(v_in, 16) && aligned(q_out, 16) && aligned(k_pool, 16) && aligned(v_pool, 16) &&
      aligned(q_norm_w, 16) && aligned(k_norm_w, 16) && q_in_stride * in_bytes % 16 == 0 &&
      k_in_stride * in_bytes % 16 == 0 && v_in_stride * in_bytes % 16 == 0 &&
      q_out_stride * out_bytes % 16 == 0;
  switch (in_dtype) {
    case PI_DTYPE_F32: return dispatch_pool<float>(p, pool_dtype, fast, stream);
    case PI_DTYPE_BF16: return dispatch_pool<__nv_bfloat16>(p, pool_dtype, fast, stream);
    case PI_DTYPE_F16: return dispatch_pool<__half>(p, pool_dtype, fast, stream);
    default: return PI_ERR_UNSUPPORTED;
  }
}
