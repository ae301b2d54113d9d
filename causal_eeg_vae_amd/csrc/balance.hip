// Balance loss of an assignment of rows to codes (or experts), the per-code counts, and its gradient:
//   p = softmax(scores);  n = rows that count;  counts_e = #{(t, j): row t counts, idx[t, j] = e};  f = counts / (n K);  P = sum_t p_t / n
//   loss = E sum_e f_e P_e;     d loss / d scores[t, e] = E / n * p_te (f_e - sum_e' f_e' p_te')          (the counts carry no gradient)
// Bound: HBM bytes - the scores are read once forward, once backward, the gradient written once.  A row lives in the registers of one lane group (1 to 64
// lanes, 16-byte loads where the rows allow them), its softmax is two butterflies; the column sums of p stay in registers over all rows
// of a wave, because a lane keeps its columns, and are joined over waves and workgroups in a fixed order: no float atomics.  The counts are
// integer LDS atomics, whose order does not matter.
// Measured, fp32, 262144 x 512, one code a row: row pass 134 us (4.0 TB/s, what a pass that only reads reaches), joins 9 + 5, gradient 189 us (5.7 TB/s).
#include "ceeg_internal.h"

namespace {
constexpr int BL_THREADS = 512;
constexpr int BL_WAVES = BL_THREADS / 64;
constexpr int BL_MAX_E = 4096;
constexpr int BL_MAX_WG = 512;
constexpr int BL_JOIN = 16;  // columns per workgroup of the join

struct BlRow {  // where the scores of a row and the columns of a lane are
  const void* s;
  int64_t ld, T;
  int E, lanes;  // lanes: lane-group size of one row, a power of two
  const uint8_t* mask;
};

// NV pieces of VEC consecutive columns per lane; piece j of lane l (of `lanes`) starts at column (j * lanes + l) * VEC
template <bool BF16, int VEC, int NV>
__device__ __forceinline__ void bl_load(const BlRow& a, int64_t t, int l, float (&x)[NV * VEC]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * a.lanes + l) * VEC;
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[j * VEC + k] = -INFINITY;
    if (c >= a.E) continue;  // VEC > 1 only where E is a multiple of it
    if (BF16) {
      const unsigned short* q = static_cast<const unsigned short*>(a.s) + t * a.ld + c;
      if (VEC == 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(q);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[j * VEC + (2 * k) % VEC] = __uint_as_float(w[k] << 16);
          x[j * VEC + (2 * k + 1) % VEC] = __uint_as_float(w[k] & 0xffff0000u);
        }
      } else {
        x[j * VEC] = ceeg_bf16_to_f32(q[0]);
      }
    } else {
      const float* q = static_cast<const float*>(a.s) + t * a.ld + c;
      if (VEC == 4) {
        const float4 u = *reinterpret_cast<const float4*>(q);
        x[j * VEC] = u.x; x[j * VEC + 1 % VEC] = u.y; x[j * VEC + 2 % VEC] = u.z; x[j * VEC + 3 % VEC] = u.w;
      } else {
        x[j * VEC] = q[0];
      }
    }
  }
}

// Over the lane group of a row, the same in each of its lanes: a whole wave joins in registers (row shifts and broadcasts end in lane 63), smaller groups by butterflies.
__device__ __forceinline__ float bl_max(int lanes, float v) {
  if (lanes == 64) {
#define BL_STEP(CTRL, ROWS) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xf, false)))
    BL_STEP(0x111, 0xf); BL_STEP(0x112, 0xf); BL_STEP(0x114, 0xf); BL_STEP(0x118, 0xf); BL_STEP(0x142, 0xa); BL_STEP(0x143, 0xc);
#undef BL_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float bl_sum(int lanes, float v) {
  if (lanes == 64) {
#define BL_STEP(CTRL, ROWS) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true))
    BL_STEP(0x111, 0xf); BL_STEP(0x112, 0xf); BL_STEP(0x114, 0xf); BL_STEP(0x118, 0xf); BL_STEP(0x142, 0xa); BL_STEP(0x143, 0xc);
#undef BL_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// x -> softmax over the lane group; a row of nothing but -inf has no probability anywhere
template <int N>
__device__ __forceinline__ void bl_softmax(int lanes, float (&x)[N]) {
  float top = x[0];
#pragma unroll
  for (int k = 1; k < N; ++k) top = fmaxf(top, x[k]);
  top = bl_max(lanes, top);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    x[k] = __expf(x[k] - base);
    sum += x[k];
  }
  sum = bl_sum(lanes, sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] *= inv;
}

struct BlOut {
  float* loss;
  int64_t* counts;
  float* stats;
};

// f = counts / (n K) of one code, NaN where a code outside [-1, E) was seen: that cannot raise an error from here, so loss and gradient say it
__device__ __forceinline__ double bl_share(long long c, double rows, int K, bool bad) {
  return bad ? __longlong_as_double(0x7ff8000000000000LL) : (double)c / (rows * K);
}

// per workgroup: part_p[wg][E] (column sums of p), part_c[wg][E] (counts), part_n[wg] = {rows that count, a code out of range was seen}.
// A grid of one workgroup (small calls, which launches would dominate) finishes by itself.
template <bool BF16, int VEC, int NV>
__global__ __launch_bounds__(BL_THREADS) void balance_rows_kernel(BlRow a, const void* __restrict__ idx, int idx64, int K, float* __restrict__ part_p,
                                                                  int32_t* __restrict__ part_c, int2* __restrict__ part_n, BlOut out) {
  extern __shared__ int s_mem[];
  int* s_c = s_mem;                                    // [E]
  float* s_p = reinterpret_cast<float*>(s_mem + a.E);  // [E]
  __shared__ int s_n[2];
  __shared__ double s_d[BL_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = threadIdx.x; e < a.E; e += BL_THREADS) s_c[e] = 0;
  if (threadIdx.x < 2) s_n[threadIdx.x] = 0;
  __syncthreads();
  const int per = 64 / a.lanes, l = lane & (a.lanes - 1), sub = lane / a.lanes;
  float acc[NV * VEC];
#pragma unroll
  for (int k = 0; k < NV * VEC; ++k) acc[k] = 0.f;
  int rows = 0, bad = 0;
  const int64_t stride = (int64_t)gridDim.x * BL_WAVES * per;
  constexpr int R = NV * VEC <= 16 ? 2 : 1;  // rows at a time: the second one's loads and butterflies run in the shadow of the first one's
  for (int64_t t0 = ((int64_t)blockIdx.x * BL_WAVES + wave) * per; t0 < a.T; t0 += R * stride) {  // the same number of turns for a wave's lanes
    float x[R][NV * VEC];
    bool on[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t t = t0 + r * stride + sub;
      on[r] = t < a.T && (!a.mask || a.mask[t]);
      if (on[r]) {
        bl_load<BF16, VEC, NV>(a, t, l, x[r]);
      } else {
#pragma unroll
        for (int k = 0; k < NV * VEC; ++k) x[r][k] = -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) bl_softmax(a.lanes, x[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t t = t0 + r * stride + sub;
#pragma unroll
      for (int k = 0; k < NV * VEC; ++k) acc[k] += x[r][k];
      if (on[r]) {
        for (int j = l; j < K; j += a.lanes) {
          const int64_t e = idx64 ? static_cast<const int64_t*>(idx)[t * K + j] : (int64_t)static_cast<const int32_t*>(idx)[t * K + j];
          if (e >= 0 && e < a.E) atomicAdd(&s_c[e], 1);
          else if (e != -1) bad = 1;
        }
        rows += l == 0;
      }
    }
  }
  // the lane groups of a wave hold the same columns
  for (int o = a.lanes; o < 64; o <<= 1) {
#pragma unroll
    for (int k = 0; k < NV * VEC; ++k) acc[k] += __shfl_xor(acc[k], o, 64);
  }
  for (int w = 0; w < BL_WAVES; ++w) {  // the waves add their sums in turn
    if (wave == w && sub == 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const int c = (j * a.lanes + l) * VEC + k;
          if (c < a.E) s_p[c] = w == 0 ? acc[j * VEC + k] : s_p[c] + acc[j * VEC + k];
        }
      }
    }
    __syncthreads();
  }
  if (rows) atomicAdd(&s_n[0], rows);
  if (bad) atomicOr(&s_n[1], 1);
  __syncthreads();
  if (gridDim.x == 1) {
    const double n = s_n[0] > 0 ? (double)s_n[0] : 1.0;
    double d = 0.0;
    for (int e = threadIdx.x; e < a.E; e += BL_THREADS) {
      const double f = bl_share(s_c[e], n, K, s_n[1] != 0);
      out.counts[e] = s_c[e];
      out.stats[e] = (float)f;
      d += f * ((double)s_p[e] / n);
    }
    d = ceeg_wave_sum_d(d);
    if (lane == 0) s_d[wave] = d;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < BL_WAVES; ++w) d += s_d[w];
      out.stats[a.E] = (float)n;
      out.loss[0] = (float)(d * a.E);
    }
    return;
  }
  for (int e = threadIdx.x; e < a.E; e += BL_THREADS) {
    part_p[(int64_t)blockIdx.x * a.E + e] = s_p[e];
    part_c[(int64_t)blockIdx.x * a.E + e] = s_c[e];
  }
  if (threadIdx.x == 0) part_n[blockIdx.x] = make_int2(s_n[0], s_n[1]);
}

// 16 columns per workgroup: P and counts over all workgroups of the row pass; f = counts / (n K); stats = [f (E), n]; dots[wg] = sum f P.  The partial sums come from other
// XCDs' memory side, so that latency bounds this: 64 threads a column, 8 loads of each in flight.
__global__ __launch_bounds__(1024) void balance_join_kernel(const float* __restrict__ part_p, const int32_t* __restrict__ part_c,
                                                            const int2* __restrict__ part_n, int wgs, int E, int K, int64_t* __restrict__ counts,
                                                            float* __restrict__ stats, double* __restrict__ dots) {
  constexpr int ROWS = 1024 / BL_JOIN;
  __shared__ double s_p[ROWS][BL_JOIN];
  __shared__ long long s_c[ROWS][BL_JOIN];
  __shared__ long long s_n[16];
  __shared__ int s_bad;
  const int col = threadIdx.x % BL_JOIN, row = threadIdx.x / BL_JOIN;
  const int e = blockIdx.x * BL_JOIN + col;
  if (threadIdx.x == 0) s_bad = 0;
  double p = 0.0;
  long long c = 0, n = 0;
  int bad = 0;
  if (e < E) {
    for (int b0 = row; b0 < wgs; b0 += 8 * ROWS) {
      float vp[8];
      int vc[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int b = b0 + ROWS * k;
        vp[k] = b < wgs ? part_p[(int64_t)b * E + e] : 0.f;
        vc[k] = b < wgs ? part_c[(int64_t)b * E + e] : 0;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        p += (double)vp[k];
        c += vc[k];
      }
    }
  }
  for (int b = threadIdx.x; b < wgs; b += 1024) {
    n += part_n[b].x;
    bad |= part_n[b].y;
  }
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  s_p[row][col] = p;
  s_c[row][col] = c;
  if ((threadIdx.x & 63) == 0) s_n[threadIdx.x >> 6] = n;
  __syncthreads();
  if (bad) s_bad = 1;  // every writer writes the same
  __syncthreads();
  if (threadIdx.x < 64) {
    p = 0.0; c = 0; n = 0;
    for (int k = 0; k < ROWS; ++k) { p += s_p[k][col]; c += s_c[k][col]; }
    for (int k = 0; k < 16; ++k) n += s_n[k];
    const double rows = n > 0 ? (double)n : 1.0;  // no row that counts: loss and gradient are zero
    const double f = bl_share(c, rows, K, s_bad != 0);
    double d = 0.0;
    if (row == 0 && e < E) {
      counts[e] = c;
      stats[e] = (float)f;
      d = f * (p / rows);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) stats[E] = (float)rows;
    d = ceeg_wave_sum_d(d);
    if (threadIdx.x == 0) dots[blockIdx.x] = d;
  }
}

__global__ void balance_loss_kernel(const double* __restrict__ dots, int n, int E, float* __restrict__ loss) {
  double d = 0.0;
  for (int k = threadIdx.x; k < n; k += 64) d += dots[k];
  d = ceeg_wave_sum_d(d);
  if (threadIdx.x == 0) loss[0] = (float)(d * E);
}

template <bool BF16, int VEC, int NV>
__global__ __launch_bounds__(BL_THREADS) void balance_grad_kernel(BlRow a, const float* __restrict__ stats, const float* __restrict__ g, void* __restrict__ ds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = 64 / a.lanes, l = lane & (a.lanes - 1), sub = lane / a.lanes;
  float f[NV * VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = (j * a.lanes + l) * VEC + k;
      f[j * VEC + k] = c < a.E ? stats[c] : 0.f;
    }
  }
  const float scale = (float)((double)g[0] * a.E / (double)stats[a.E]);
  const int64_t stride = (int64_t)gridDim.x * BL_WAVES * per;
  for (int64_t t0 = ((int64_t)blockIdx.x * BL_WAVES + wave) * per; t0 < a.T; t0 += stride) {
    const int64_t t = t0 + sub;
    if (t >= a.T) continue;  // whole lane groups leave together; the butterflies stay inside a group
    const bool on = !a.mask || a.mask[t];
    float x[NV * VEC];
    if (on) {
      bl_load<BF16, VEC, NV>(a, t, l, x);
      bl_softmax(a.lanes, x);
      float d = 0.f;
#pragma unroll
      for (int k = 0; k < NV * VEC; ++k) d = __fmaf_rn(f[k], x[k], d);
      d = bl_sum(a.lanes, d);
#pragma unroll
      for (int k = 0; k < NV * VEC; ++k) x[k] = scale * x[k] * (f[k] - d);
    } else {
#pragma unroll
      for (int k = 0; k < NV * VEC; ++k) x[k] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * a.lanes + l) * VEC;
      if (c >= a.E) continue;
      if (BF16) {
        unsigned short* q = static_cast<unsigned short*>(ds) + t * a.E + c;
        if (VEC == 8) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = (uint32_t)ceeg_f32_to_bf16(x[j * VEC + (2 * k) % VEC]) | ((uint32_t)ceeg_f32_to_bf16(x[j * VEC + (2 * k + 1) % VEC]) << 16);
          *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          q[0] = ceeg_f32_to_bf16(x[j * VEC]);
        }
      } else {
        float* q = static_cast<float*>(ds) + t * a.E + c;
        if (VEC == 4) *reinterpret_cast<float4*>(q) = make_float4(x[j * VEC], x[j * VEC + 1 % VEC], x[j * VEC + 2 % VEC], x[j * VEC + 3 % VEC]);
        else q[0] = x[j * VEC];
      }
    }
  }
}

// lanes of a row and pieces per lane: the fewest lanes that hold a row in one piece each, 64 with as many pieces as it takes beyond that
void bl_shape(int E, int vec, int* lanes, int* nv) {
  const int pieces = (E + vec - 1) / vec;
  int l = 1;
  while (l < 64 && l < pieces) l <<= 1;
  *lanes = l;
  *nv = (pieces + l - 1) / l;
}
bool bl_vec(const void* s, int64_t ld, int E, int dtype) {
  const int per = dtype == CEEG_BF16 ? 8 : 4;
  return E % per == 0 && ld % per == 0 && ceeg_aligned(s, 16);
}
int bl_wgs(int64_t T, int E, int lanes) {
  // as many workgroups as there are rows for, 512 at most (16 waves per compute unit; 131072 x 256: 51 us, 256 workgroups 74, 1024 54), half of that where their partial sums
  // would weigh more than the rows (65536 x 4096: 220 us, 512 workgroups 249; 131072 x 1024 the other way round, 133 and 110)
  int64_t wgs = (T + BL_WAVES * (64 / lanes) - 1) / (BL_WAVES * (64 / lanes));
  const int64_t cap = E > 1024 ? BL_MAX_WG / 2 : BL_MAX_WG;
  return (int)(wgs < cap ? wgs : cap);
}
int bl_check(const void* s, int64_t ld, int64_t T, int E, int dtype) {
  if (T < 1 || T > ((int64_t)1 << 31) - 1 || E < 1 || ld < E || !s) return CEEG_EINVAL;
  if (dtype != CEEG_F32 && dtype != CEEG_BF16) return CEEG_EUNSUPPORTED;
  if (E > BL_MAX_E) return CEEG_EUNSUPPORTED;
  if (!ceeg_aligned(s, dtype == CEEG_F32 ? 4 : 2)) return CEEG_EINVAL;
  return CEEG_OK;
}
}  // namespace

#define BL_DISPATCH(KERNEL, ...)                                                          \
  do {                                                                                    \
    if (dtype == CEEG_F32) {                                                              \
      if (vec == 4) {                                                                     \
        if (nv <= 1) KERNEL<false, 4, 1> __VA_ARGS__;                                     \
        else if (nv <= 2) KERNEL<false, 4, 2> __VA_ARGS__;                                \
        else if (nv <= 4) KERNEL<false, 4, 4> __VA_ARGS__;                                \
        else KERNEL<false, 4, 16> __VA_ARGS__;                                            \
      } else {                                                                            \
        if (nv <= 1) KERNEL<false, 1, 1> __VA_ARGS__;                                     \
        else if (nv <= 4) KERNEL<false, 1, 4> __VA_ARGS__;                                \
        else if (nv <= 16) KERNEL<false, 1, 16> __VA_ARGS__;                              \
        else KERNEL<false, 1, 64> __VA_ARGS__;                                            \
      }                                                                                   \
    } else {                                                                              \
      if (vec == 8) {                                                                     \
        if (nv <= 1) KERNEL<true, 8, 1> __VA_ARGS__;                                      \
        else if (nv <= 2) KERNEL<true, 8, 2> __VA_ARGS__;                                 \
        else KERNEL<true, 8, 8> __VA_ARGS__;                                              \
      } else {                                                                            \
        if (nv <= 1) KERNEL<true, 1, 1> __VA_ARGS__;                                      \
        else if (nv <= 4) KERNEL<true, 1, 4> __VA_ARGS__;                                 \
        else if (nv <= 16) KERNEL<true, 1, 16> __VA_ARGS__;                               \
        else KERNEL<true, 1, 64> __VA_ARGS__;                                             \
      }                                                                                   \
    }                                                                                     \
  } while (0)

extern "C" size_t ceeg_balance_ws_bytes(int64_t T, int E) {
  if (T < 1 || E < 1 || E > BL_MAX_E) return 0;
  int lanes, nv;
  bl_shape(E, 1, &lanes, &nv);  // one column a piece has the most lanes per row, hence the most workgroups
  const size_t wgs = (size_t)bl_wgs(T, E, lanes);
  return ceeg_ws_part(wgs * E, 4) + ceeg_ws_part(wgs * E, 4) + ceeg_ws_part(wgs, 8) + ceeg_ws_part(BL_MAX_E / BL_JOIN, 8);
}

extern "C" int ceeg_balance_fwd(const void* scores, int64_t ld, int dtype, const void* idx, int idx_bytes, int64_t T, int E, int K, const uint8_t* mask,
                                float* loss, int64_t* counts, float* stats, void* ws, size_t ws_bytes, void* stream) {
  const int rc = bl_check(scores, ld, T, E, dtype);
  if (rc) return rc;
  if (K < 1 || K > E || !idx || !loss || !counts || !stats || (idx_bytes != 4 && idx_bytes != 8) || !ceeg_aligned(idx, idx_bytes)) return CEEG_EINVAL;
  if (T > ((int64_t)1 << 38) / K) return CEEG_EUNSUPPORTED;  // a workgroup's counts are 32 bits
  if (!ws || ws_bytes < ceeg_balance_ws_bytes(T, E) || !ceeg_aligned(ws, 256)) return CEEG_EWORKSPACE;
  const int vec = bl_vec(scores, ld, E, dtype) ? (dtype == CEEG_BF16 ? 8 : 4) : 1;
  BlRow a{scores, ld, T, E, 0, mask};
  int nv;
  bl_shape(E, vec, &a.lanes, &nv);
  const int wgs = bl_wgs(T, E, a.lanes);
  CeegWs w(ws, ws_bytes);
  float* part_p = w.take<float>((size_t)wgs * E);
  int32_t* part_c = w.take<int32_t>((size_t)wgs * E);
  int2* part_n = w.take<int2>(wgs);
  double* dots = w.take<double>(BL_MAX_E / BL_JOIN);
  if (!w.ok) return CEEG_EWORKSPACE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t lds = (size_t)E * 8;  // 32 KB at most
  BL_DISPATCH(balance_rows_kernel, <<<wgs, BL_THREADS, lds, st>>>(a, idx, idx_bytes == 8, K, part_p, part_c, part_n, BlOut{loss, counts, stats}));
  CEEG_CHECK_LAUNCH();
  if (wgs == 1) return CEEG_OK;
  const int joins = (E + BL_JOIN - 1) / BL_JOIN;
  balance_join_kernel<<<joins, 1024, 0, st>>>(part_p, part_c, part_n, wgs, E, K, counts, stats, dots);
  CEEG_CHECK_LAUNCH();
  balance_loss_kernel<<<1, 64, 0, st>>>(dots, joins, E, loss);
  CEEG_CHECK_LAUNCH();
  return CEEG_OK;
}

extern "C" int ceeg_balance_bwd(const void* scores, int64_t ld, int dtype, int64_t T, int E, const uint8_t* mask, const float* stats, const float* g,
                                void* dscores, void* stream) {
  const int rc = bl_check(scores, ld, T, E, dtype);
  if (rc) return rc;
  if (!stats || !g || !dscores || !ceeg_aligned(dscores, 16)) return CEEG_EINVAL;
  const int vec = bl_vec(scores, ld, E, dtype) ? (dtype == CEEG_BF16 ? 8 : 4) : 1;
  BlRow a{scores, ld, T, E, 0, mask};
  int nv;
  bl_shape(E, vec, &a.lanes, &nv);
  const int64_t units = (T + BL_WAVES * (64 / a.lanes) - 1) / (BL_WAVES * (64 / a.lanes));
  const unsigned wgs = (unsigned)(units < 1024 ? units : 1024);  // four per compute unit: every lane reads its f once for many rows (2048 to 8192: 3 % either way)
  const hipStream_t st = static_cast<hipStream_t>(stream);
  BL_DISPATCH(balance_grad_kernel, <<<wgs, BL_THREADS, 0, st>>>(a, stats, g, dscores));
  CEEG_CHECK_LAUNCH();
  return CEEG_OK;
}
