// AdamW over a list of tensors in one launch, first and second moment in 32 bits or in 8:
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2;   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
// 8 bits: m and sqrt(v) (the root halves the range of exponents that has to fit) are e4m3 numbers times one fp32 scale per 256 consecutive elements, the
// block's largest magnitude / 448.  A step changes v by 1 - b2 of itself, far less than half a step of an 8-bit number, so rounding to
// nearest would hold v where it is for ever; a magnitude is therefore rounded UP with the probability of what rounding down leaves out, which keeps the
// expectation of m and of sqrt(v), what the update divides by.  v itself, the root's square, comes out larger by the rounding's variance: 4 % of v once it has
// settled, and the root 0.8 % (normal gradients, b2 = 0.99 and 0.999 alike).
// 16 random bits of Philox per value.  sqrt(v) > 0 never becomes 0: a denominator that vanishes while m does not would blow the next step up.
// Bound: HBM bytes (fp32 28 per element; 8 bits 16 with fp32 parameters, 10 with bf16).  A wave takes one block of 256 elements, 4 per lane - 16-byte loads, the
// block's maximum by one butterfly, one Philox call per lane for its four elements - so the 8-bit form needs no LDS and no barrier.
// Measured, 66 M elements in 148 tensors: 32 bits 347 us (5.3 TB/s); 8 bits 238 us (4.4 TB/s: vector instructions, about 120 an element, are as long as the bytes), with 50 M
// bf16 parameters 145 us (3.5 TB/s; 130 instructions).
// The tensors' pointers travel in the kernel arguments: no table in device memory, nothing to copy or to keep alive.
#include <math.h>
#include "ceeg_internal.h"

namespace {
constexpr int AW_THREADS = 256;
constexpr int AW_BLOCK = 256;   // elements per wave step and per 8-bit scale
constexpr int AW_LIST = 56;     // tensors per launch: 56 * 60 + 80 bytes stay below the 4096 bytes of kernel arguments
constexpr float AW_TOP = 448.f; // largest e4m3 number
constexpr float AW_PER_TOP = 1.f / 448.f;
constexpr float AW_TINY = 0x1p-100f;

struct AwList {
  void* p[AW_LIST];
  const void* g[AW_LIST];
  void* m[AW_LIST];
  void* v[AW_LIST];
  float* ms[AW_LIST];
  float* vs[AW_LIST];
  int64_t n[AW_LIST];
  uint32_t first[AW_LIST];  // first workgroup of the tensor
  int32_t count;
};
struct AwHyper {
  float b1, b2, omb1, omb2, eps, decay, step_size, inv_sqrt_c2;
  double b1d, b2d, lrd, wdd;
  const float* step_dev;  // NULL: step_size and inv_sqrt_c2 above hold
  const float* lr_dev;    // NULL: lrd
  uint64_t seed;
  uint32_t ordinal;       // place of the launch's first tensor in the caller's list
  uint32_t per_wg;        // elements per workgroup
};

template <bool FULL, bool BF16>
__device__ __forceinline__ void aw_load4(const void* p, int64_t i, int64_t n, bool vec, float (&x)[4]) {
  if (BF16) {
    const unsigned short* q = static_cast<const unsigned short*>(p) + i;
    if (FULL || (vec && i + 4 <= n)) {
      const ushort4 u = *reinterpret_cast<const ushort4*>(q);
      x[0] = ceeg_bf16_to_f32(u.x); x[1] = ceeg_bf16_to_f32(u.y); x[2] = ceeg_bf16_to_f32(u.z); x[3] = ceeg_bf16_to_f32(u.w);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = i + k < n ? ceeg_bf16_to_f32(q[k]) : 0.f;
    }
  } else {
    const float* q = static_cast<const float*>(p) + i;
    if (FULL || (vec && i + 4 <= n)) {
      const float4 u = *reinterpret_cast<const float4*>(q);
      x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = i + k < n ? q[k] : 0.f;
    }
  }
}
template <bool FULL, bool BF16>
__device__ __forceinline__ void aw_store4(void* p, int64_t i, int64_t n, bool vec, const float (&x)[4]) {
  if (BF16) {  // a bf16 parameter is rounded to nearest, as every bf16 result of this library
    unsigned short* q = static_cast<unsigned short*>(p) + i;
    if (FULL || (vec && i + 4 <= n)) {
      *reinterpret_cast<ushort4*>(q) = make_ushort4(ceeg_f32_to_bf16(x[0]), ceeg_f32_to_bf16(x[1]), ceeg_f32_to_bf16(x[2]), ceeg_f32_to_bf16(x[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) q[k] = ceeg_f32_to_bf16(x[k]);
    }
  } else {
    float* q = static_cast<float*>(p) + i;
    if (FULL || (vec && i + 4 <= n)) {
      *reinterpret_cast<float4*>(q) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) q[k] = x[k];
    }
  }
}
template <bool FULL>
__device__ __forceinline__ uint32_t aw_codes4(const uint8_t* p, int64_t i, int64_t n, bool vec) {
  if (FULL || (vec && i + 4 <= n)) return *reinterpret_cast<const uint32_t*>(p + i);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) w |= (uint32_t)p[i + k] << (8 * k);
  return w;
}
template <bool FULL>
__device__ __forceinline__ void aw_put_codes4(uint8_t* p, int64_t i, int64_t n, bool vec, uint32_t w) {
  if (FULL || (vec && i + 4 <= n)) {
    *reinterpret_cast<uint32_t*>(p + i) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = (uint8_t)(w >> (8 * k));
  }
}
// ceeg_philox with each 32 x 32 product as one 64-bit instruction
__device__ __forceinline__ uint4 aw_philox(uint64_t seed, uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) {
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0; c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1; c3 = (uint32_t)a;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ bool aw_finite(float x) { return fabsf(x) <= 3.402823466e38f; }
// the largest of 64 lanes' values >= 0, the same in every lane: six steps in registers
__device__ __forceinline__ float aw_wave_max(int x) {  // bits of values >= 0: the larger value has the larger bits, infinities and NaN the largest
#define AW_MAX(CTRL, ROWS) x = max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, true))
  AW_MAX(0x111, 0xf);  // row_shr 1, 2, 4, 8: lane 15 of each row of 16
  AW_MAX(0x112, 0xf);
  AW_MAX(0x114, 0xf);
  AW_MAX(0x118, 0xf);
  AW_MAX(0x142, 0xa);  // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3: lane 63
  AW_MAX(0x143, 0xc);
#undef AW_MAX
  return __int_as_float(__builtin_amdgcn_readlane(x, 63));
}
// b^t by squaring: t 2^-53 of itself off at most, and so 1 - b^t >= (1 - b) t b^t no more than 2^-53 / (1 - b) of itself
__device__ __forceinline__ double aw_power(double b, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1u) r *= b;
  return r;
}
// 1 / b for b and 1 / b of ordinary size (a block's scale lies between 2^-109 and 2^120), nearly rounded: one Newton step behind the instruction
__device__ __forceinline__ float aw_reciprocal(float b) {
  const float r = __builtin_amdgcn_rcpf(b);
  return __fmaf_rn(__fmaf_rn(-b, r, 1.f), r, r);
}
// a / b, correctly rounded, from the (nearly) rounded reciprocal r of b: a quotient within a unit and one exact remainder
__device__ __forceinline__ float aw_quotient(float a, float b, float r) {
  const float q = a * r;
  return __fmaf_rn(__fmaf_rn(-q, b, a), r, q);
}
// x / scale as an e4m3 number, rounded by the 16 random bits `rnd` so that the expectation of its magnitude is kept.  per_scale: 1 / scale, 0 where the scale is.
// SECOND: a magnitude > 0 does not become 0.
template <bool SECOND, bool FINITE>
__device__ __forceinline__ uint32_t aw_round(float x, float scale, float per_scale, float rnd) {
  const float a = fabsf(x), y = fminf(aw_quotient(a, scale, per_scale), AW_TOP);
  const uint32_t u = __float_as_uint(y);
  const bool small = y < 0x1p-6f;  // there the numbers are 2^-9 apart
  const float t = y * 512.f, below = floorf(t);
  const float share = small ? t - below : (float)(u & 0xfffffu) * 0x1p-20f;
  uint32_t c = small ? (uint32_t)below : (u >> 20) - (120u << 3);
  c += share * 65536.f + rnd >= 65536.f;
  if (SECOND && c == 0u && y > 0.f) c = 1u;
  if (!FINITE && !aw_finite(x)) c = 0x7fu;  // stays a NaN
  return c | (__float_as_uint(x) >> 24 & 0x80u);
}

template <bool B> struct AwBool { static constexpr bool value = B; };

template <bool BF16, int BITS>
__global__ __launch_bounds__(AW_THREADS) void adamw_kernel(AwList L, AwHyper h) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int lo = 0, hi = L.count - 1;  // the tensor whose workgroups hold this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const int64_t n = L.n[lo];
  const int64_t begin = (int64_t)(blockIdx.x - L.first[lo]) * h.per_wg;
  const int64_t end = begin + h.per_wg < n ? begin + h.per_wg : n;
  float step_size = h.step_size, inv_sqrt_c2 = h.inv_sqrt_c2, decay = h.decay;
  uint64_t seed = h.seed;
  if (h.step_dev || h.lr_dev) {  // one wave finds the factors: in 64 bits they cost as much as half a block of elements
    __shared__ float s_factor[3];
    if (wave == 0) {
      const double lr = h.lr_dev ? (double)h.lr_dev[0] : h.lrd;
      float size = (float)(lr * h.b1d), inv = inv_sqrt_c2;  // without step_dev: the host put 1 / (1 - b1^t) there
      if (h.step_dev) {
        const uint32_t t = (uint32_t)h.step_dev[0];  // whole, and below 2^24 where it can still be counted up
        size = (float)(lr / (1.0 - aw_power(h.b1d, t)));
        inv = (float)(1.0 / sqrt(1.0 - aw_power(h.b2d, t)));
      }
      if (lane == 0) {
        s_factor[0] = size;
        s_factor[1] = inv;
        s_factor[2] = (float)(1.0 - lr * h.wdd);
      }
    }
    __syncthreads();
    step_size = s_factor[0];
    inv_sqrt_c2 = s_factor[1];
    decay = s_factor[2];
    if (h.step_dev) seed += (uint64_t)(int64_t)h.step_dev[0] * 0x9E3779B97F4A7C15ull;  // a replayed launch draws other numbers every step
  }
  void* const p = L.p[lo];
  const void* const g = L.g[lo];
  void* const m = L.m[lo];
  void* const v = L.v[lo];
  const uintptr_t pg = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g);
  const uintptr_t mv = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
  const bool vec = (pg & (BF16 ? 7 : 15)) == 0, svec = (mv & (BITS == 8 ? 3 : 15)) == 0;

  // FULL: a block of 256 elements on aligned addresses, without a check per element
  auto block = [&](auto full, int64_t b0) {
    constexpr bool FULL = decltype(full)::value;
    const int64_t i = b0 + 4 * lane;
    float pv[4], gv[4], mo[4], vo[4], root[4];
    aw_load4<FULL, BF16>(p, i, n, vec, pv);
    aw_load4<FULL, BF16>(g, i, n, vec, gv);
    if (BITS == 8) {
      const float sm = L.ms[lo][b0 / AW_BLOCK], sv = L.vs[lo][b0 / AW_BLOCK];
      const uint32_t cm = aw_codes4<FULL>(static_cast<const uint8_t*>(m), i, n, svec), cv = aw_codes4<FULL>(static_cast<const uint8_t*>(v), i, n, svec);
      mo[0] = __builtin_amdgcn_cvt_f32_fp8(cm, 0); mo[1] = __builtin_amdgcn_cvt_f32_fp8(cm, 1);
      mo[2] = __builtin_amdgcn_cvt_f32_fp8(cm, 2); mo[3] = __builtin_amdgcn_cvt_f32_fp8(cm, 3);
      root[0] = __builtin_amdgcn_cvt_f32_fp8(cv, 0); root[1] = __builtin_amdgcn_cvt_f32_fp8(cv, 1);
      root[2] = __builtin_amdgcn_cvt_f32_fp8(cv, 2); root[3] = __builtin_amdgcn_cvt_f32_fp8(cv, 3);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float u = root[k] * sv;
        mo[k] *= sm;
        vo[k] = u * u;
      }
    } else {
      aw_load4<FULL, false>(m, i, n, svec, mo);
      aw_load4<FULL, false>(v, i, n, svec, vo);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mo[k] = h.b1 * mo[k] + h.omb1 * gv[k];
      vo[k] = h.b2 * vo[k] + h.omb2 * (gv[k] * gv[k]);
      root[k] = sqrtf(vo[k]);
      // the reciprocal by the instruction alone, a unit (2^-23) off at most: of an update, which is itself lr of a parameter of ordinary size
      pv[k] = pv[k] * decay - step_size * (mo[k] * __builtin_amdgcn_rcpf(root[k] * inv_sqrt_c2 + h.eps));
    }
    aw_store4<FULL, BF16>(p, i, n, vec, pv);
    if (BITS == 32) {
      aw_store4<FULL, false>(m, i, n, svec, mo);
      aw_store4<FULL, false>(v, i, n, svec, vo);
      return;
    }
    int bm = 0, bv = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!FULL && i + k >= n) mo[k] = root[k] = 0.f;
      bm = max(bm, __float_as_int(fabsf(mo[k])));
      bv = max(bv, __float_as_int(fabsf(root[k])));
    }
    float tm = aw_wave_max(bm), tv = aw_wave_max(bv);
    const bool finite = aw_finite(tm) && aw_finite(tv);
    if (!finite) {  // infinities and NaN do not set a block's scale
      bm = bv = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bm = max(bm, aw_finite(mo[k]) ? __float_as_int(fabsf(mo[k])) : 0);
        bv = max(bv, aw_finite(root[k]) ? __float_as_int(root[k]) : 0);
      }
      tm = aw_wave_max(bm);
      tv = aw_wave_max(bv);
    }
    const float sm = tm < AW_TINY ? 0.f : tm * AW_PER_TOP, sv = tv < AW_TINY ? 0.f : tv * AW_PER_TOP;
    const float pm = sm > 0.f ? aw_reciprocal(sm) : 0.f, pr = sv > 0.f ? aw_reciprocal(sv) : 0.f;
    const uint64_t quad = (uint64_t)i >> 2;
    const uint4 r = aw_philox(seed, (uint32_t)quad, (uint32_t)(quad >> 32), CEEG_TAG_ADAMW, h.ordinal + lo);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t cm = 0, cv = 0;
    if (finite) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        cm |= aw_round<false, true>(mo[k], sm, pm, (float)(w[k] & 0xffffu)) << (8 * k);
        cv |= aw_round<true, true>(root[k], sv, pr, (float)(w[k] >> 16)) << (8 * k);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        cm |= aw_round<false, false>(mo[k], sm, pm, (float)(w[k] & 0xffffu)) << (8 * k);
        cv |= aw_round<true, false>(root[k], sv, pr, (float)(w[k] >> 16)) << (8 * k);
      }
    }
    aw_put_codes4<FULL>(static_cast<uint8_t*>(m), i, n, svec, cm);
    aw_put_codes4<FULL>(static_cast<uint8_t*>(v), i, n, svec, cv);
    if (lane == 0) {
      L.ms[lo][b0 / AW_BLOCK] = sm;
      L.vs[lo][b0 / AW_BLOCK] = sv;
    }
  };
  for (int64_t b0 = begin + (int64_t)wave * AW_BLOCK; b0 < end; b0 += AW_THREADS / 64 * AW_BLOCK) {
    if (vec && svec && b0 + AW_BLOCK <= n) block(AwBool<true>{}, b0);
    else block(AwBool<false>{}, b0);
  }
}
}  // namespace

extern "C" int ceeg_adamw_block(void) { return AW_BLOCK; }

extern "C" int ceeg_adamw_step(int tensors, const int64_t* numel, void* const* p, const void* const* g, void* const* m, void* const* v,
                               float* const* m_scale, float* const* v_scale, int dtype, int state_bits, double lr, double beta1, double beta2,
                               double eps, double weight_decay, int64_t step, const float* lr_dev, const float* step_dev, uint64_t seed,
                               void* stream) {
  if (tensors < 0 || (tensors > 0 && (!numel || !p || !g || !m || !v))) return CEEG_EINVAL;
  if (dtype != CEEG_F32 && dtype != CEEG_BF16) return CEEG_EUNSUPPORTED;
  if (state_bits != 8 && state_bits != 32) return CEEG_EUNSUPPORTED;
  if (state_bits == 8 && tensors > 0 && (!m_scale || !v_scale)) return CEEG_EINVAL;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0) || (!step_dev && step < 1)) return CEEG_EINVAL;
  const uintptr_t palign = dtype == CEEG_F32 ? 3 : 1;
  int64_t total = 0;
  for (int t = 0; t < tensors; ++t) {
    if (numel[t] < 0 || numel[t] > ((int64_t)1 << 40)) return CEEG_EINVAL;
    if (numel[t] == 0) continue;
    if (!p[t] || !g[t] || !m[t] || !v[t] || ((reinterpret_cast<uintptr_t>(p[t]) | reinterpret_cast<uintptr_t>(g[t])) & palign)) return CEEG_EINVAL;
    if (state_bits == 8 ? (!m_scale[t] || !v_scale[t] || !ceeg_aligned(m_scale[t], 4) || !ceeg_aligned(v_scale[t], 4))
                        : (!ceeg_aligned(m[t], 4) || !ceeg_aligned(v[t], 4))) return CEEG_EINVAL;
    total += numel[t];
  }
  AwHyper h;
  const double c1 = step_dev ? 1.0 : 1.0 - pow(beta1, (double)step), c2 = step_dev ? 1.0 : 1.0 - pow(beta2, (double)step);
  h.b1 = (float)beta1; h.b2 = (float)beta2; h.omb1 = (float)(1.0 - beta1); h.omb2 = (float)(1.0 - beta2);
  h.eps = (float)eps; h.decay = (float)(1.0 - lr * weight_decay); h.step_size = (float)(lr / c1); h.inv_sqrt_c2 = (float)(1.0 / sqrt(c2));
  h.b1d = step_dev ? beta1 : 1.0 / c1; h.b2d = beta2; h.lrd = lr; h.wdd = weight_decay;
  h.step_dev = step_dev; h.lr_dev = lr_dev;
  h.seed = seed;
  // Elements per workgroup.  One block per wave fills the compute units soonest and balances them best (32 bits, 148 tensors of 66 M together: 352 us, 379 with 4096; 8 bits,
  // 1 M: 7.9 us instead of 9.2, 2 M 12.4 and 12.7).  The longer start of 8 bits is worth four blocks a wave from 4 M on (one tensor of 4 M: 19.6 us instead of 20.9, 8192 21.3;
  // 148 tensors of 66 M: 235 us instead of 266, 238 with 8192).
  h.per_wg = state_bits == 8 && total >= (int64_t)1 << 22 ? 4096 : 1024;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for (int t = 0; t < tensors;) {
    AwList L;
    int c = 0;
    uint64_t wgs = 0;
    h.ordinal = (uint32_t)t;
    // a launch takes consecutive tensors (empty ones keep their place) while their workgroups fit a grid
    for (; t < tensors && c < AW_LIST; ++t, ++c) {
      const uint64_t more = (uint64_t)((numel[t] + h.per_wg - 1) / h.per_wg);
      if (more > 0x7fffffffull) return CEEG_EUNSUPPORTED;
      if (wgs + more > 0x7fffffffull) break;
      L.p[c] = p[t]; L.g[c] = g[t]; L.m[c] = m[t]; L.v[c] = v[t]; L.n[c] = numel[t]; L.first[c] = (uint32_t)wgs;
      L.ms[c] = state_bits == 8 ? m_scale[t] : nullptr;
      L.vs[c] = state_bits == 8 ? v_scale[t] : nullptr;
      wgs += more;
    }
    L.count = c;
    for (int k = c; k < AW_LIST; ++k) { L.p[k] = L.m[k] = L.v[k] = nullptr; L.g[k] = nullptr; L.ms[k] = L.vs[k] = nullptr; L.n[k] = 0; L.first[k] = 0; }
    if (wgs == 0) continue;
    const dim3 grid((unsigned)wgs), block(AW_THREADS);
    if (dtype == CEEG_F32) {
      if (state_bits == 32) adamw_kernel<false, 32><<<grid, block, 0, st>>>(L, h);
      else adamw_kernel<false, 8><<<grid, block, 0, st>>>(L, h);
    } else {
      if (state_bits == 32) adamw_kernel<true, 32><<<grid, block, 0, st>>>(L, h);
      else adamw_kernel<true, 8><<<grid, block, 0, st>>>(L, h);
    }
    CEEG_CHECK_LAUNCH();
  }
  return CEEG_OK;
}
