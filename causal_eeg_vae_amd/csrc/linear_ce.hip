// Softmax cross entropy behind a vocabulary product, and its gradient, without the logits in memory:
//   l_tv = <h_t, W_v>;   lse_t = log sum_v exp l_tv;   loss_t = lse_t - l_t,y(t);   dl_tv = r_t (exp(l_tv - lse_t) - [v = y(t)])
//   dh = s dl W;   dW = s dl^T h;      s r_t = what comes back for loss_t (r = 1 for every token of a mean or a sum)
// Bound: the matrix cores (2 T H V operations forward, 6 T H V more backward: the logits are computed again, which costs less than
// writing them and reading them back).  Everything runs on bf16 tiles (v_mfma_f32_16x16x32_bf16, fp32 accumulators):
//   bf16 inputs  one plane each;
//   fp32 inputs  three bf16 planes each (8 bits of the mantissa each) and the six products whose terms reach 2^-24 of the result,
//                small ones first - 6/16 of the bf16 rate instead of the 1/16 of the fp32 instruction.
// Tokens that are ignored are dropped before the first product: their rows are packed away, the grids cover all T tokens and what
// lies behind the last one that counts leaves at once (its number is read on the device, the host never waits for it).
// The vocabulary is taken in pieces; of a piece only dl is held (bf16, as it is and transposed), so that every product reads both
// operands along its summed axis.  No float atomics: the pieces of a sum are added in a fixed order.
#include "ceeg_internal.h"

namespace {
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;

constexpr int BK = 64;                                   // elements of the summed axis per LDS tile
constexpr int64_t CE_CAP = (int64_t)1 << 30;             // bytes that the pieces of the backward pass may take together
constexpr int64_t CE_MAX_PIECE = (int64_t)1 << 20;       // columns per piece: 32-bit offsets inside a tile
// planes of A and B in the products (2,0) (0,2) (1,1) | (1,0) (0,1) | (0,0), two bits each; a bar is a factor of 2^-8 on what is summed so far
constexpr unsigned CE_PAIRS_A = 2u | 0u << 2 | 1u << 4 | 1u << 6 | 0u << 8 | 0u << 10;
constexpr unsigned CE_PAIRS_B = 0u | 2u << 2 | 1u << 4 | 0u << 6 | 1u << 8 | 0u << 10;

// x = p[0] + 2^-8 p[1] + 2^-16 p[2], each rounded to nearest.  Without the powers of two the lower planes of a small x would fall below what bf16
// holds (2^-133); with them every fp32 number, subnormal ones too, is held to its last bit.  What rounds past the largest bf16 number is cut
// instead; what is not finite stays in the first plane.
__device__ __forceinline__ unsigned short ce_plane(float x) {
  const float a = fabsf(x);
  return a >= 3.3961775e38f && a <= 3.402823466e38f ? (unsigned short)(__float_as_uint(x) >> 16) : ceeg_f32_to_bf16(x);
}
__device__ __forceinline__ void ce_split(float x, unsigned short (&p)[3]) {
  p[0] = ce_plane(x);
  const float r1 = fabsf(x) <= 3.402823466e38f ? (x - ceeg_bf16_to_f32(p[0])) * 256.f : 0.f;
  p[1] = ce_plane(r1);
  p[2] = ce_plane((r1 - ceeg_bf16_to_f32(p[1])) * 256.f);
}

// ------------------------------------------------------------------------------------------------ which tokens count
// One workgroup: rows[j] = j-th token that counts, pos[t] = j or -1, yc[j] = its class (-1: outside [0, V)), n[0] = how many.
__global__ __launch_bounds__(1024) void ce_tokens_kernel(const int64_t* __restrict__ y, int64_t T, int64_t V, int64_t ignore, int32_t* __restrict__ n,
                                                         int32_t* __restrict__ rows, int32_t* __restrict__ pos, int32_t* __restrict__ yc) {
  __shared__ int s_sum[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int64_t t0 = 0; t0 < T; t0 += 4096) {
    const int64_t t = t0 + 4 * threadIdx.x;
    int64_t v[4];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = t + k < T ? y[t + k] : ignore;
      mine += v[k] != ignore;
    }
    int pre = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(pre, o, 64);
      if (lane >= o) pre += u;
    }
    if (lane == 63) s_sum[wave] = pre;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? s_sum[w] : 0;
      all += s_sum[w];
    }
    int j = base + before + pre - mine;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (t + k >= T) continue;
      if (v[k] != ignore) {
        rows[j] = (int32_t)(t + k);
        yc[j] = v[k] >= 0 && v[k] < V ? (int32_t)v[k] : -1;
        pos[t + k] = j++;
      } else {
        pos[t + k] = -1;
      }
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) n[0] = base;
}

// ------------------------------------------------------------------------------------------------ planes
// 64 x 64 tiles of a row-major [R, C] matrix (rows taken through `rows` where given, R from the device where `count` is given)
//   -> planes row by row [P][*][Cp] (`out`, columns C..Cp zero) and / or transposed [P][C][Rp] (`outT`, rows R.. to the next multiple of 64 zero)
template <bool F32>
__global__ __launch_bounds__(256) void ce_pack_kernel(const void* __restrict__ src, int64_t ld, const int32_t* __restrict__ rows,
                                                      const int32_t* __restrict__ count, int R, int C, unsigned short* __restrict__ out, int64_t plane, int Cp,
                                                      unsigned short* __restrict__ outT, int64_t planeT, int64_t Rp) {
  __shared__ float s_t[64][65];
  const int n = count ? count[0] : R;
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
  if (r0 >= n) return;
  const int cq = (threadIdx.x & 15) * 4, rr = threadIdx.x >> 4;
  const bool vec = (ld & 3) == 0 && (reinterpret_cast<uintptr_t>(src) & (F32 ? 15 : 7)) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + rr + 16 * i, c = c0 + cq;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < n) {
      const int64_t at = (rows ? (int64_t)rows[r] : (int64_t)r) * ld + c;
      if (F32) {
        const float* q = static_cast<const float*>(src) + at;
        if (vec && c + 4 <= C) {
          const float4 u = *reinterpret_cast<const float4*>(q);
          x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = c + k < C ? q[k] : 0.f;
        }
      } else {
        const unsigned short* q = static_cast<const unsigned short*>(src) + at;
        if (vec && c + 4 <= C) {
          const ushort4 u = *reinterpret_cast<const ushort4*>(q);
          x[0] = ceeg_bf16_to_f32(u.x); x[1] = ceeg_bf16_to_f32(u.y); x[2] = ceeg_bf16_to_f32(u.z); x[3] = ceeg_bf16_to_f32(u.w);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = c + k < C ? ceeg_bf16_to_f32(q[k]) : 0.f;
        }
      }
    }
    if (out && r < n) {
      unsigned short p[4][3];
#pragma unroll
      for (int k = 0; k < 4; ++k) ce_split(x[k], p[k]);
#pragma unroll
      for (int a = 0; a < (F32 ? 3 : 1); ++a)
        *reinterpret_cast<ushort4*>(out + a * plane + (int64_t)r * Cp + c) = make_ushort4(p[0][a], p[1][a], p[2][a], p[3][a]);
    }
    if (outT) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s_t[rr + 16 * i][cq + k] = x[k];
    }
  }
  if (!outT) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + rr + 16 * i;
    if (c >= C) continue;
    unsigned short p[4][3];
#pragma unroll
    for (int k = 0; k < 4; ++k) ce_split(s_t[cq + k][rr + 16 * i], p[k]);
#pragma unroll
    for (int a = 0; a < (F32 ? 3 : 1); ++a)
      *reinterpret_cast<ushort4*>(outT + a * planeT + (int64_t)c * Rp + r0 + cq) = make_ushort4(p[0][a], p[1][a], p[2][a], p[3][a]);
  }
}

// ------------------------------------------------------------------------------------------------ products
// C[n][m] = sum over pairs of planes, over k: A[m][k] B[n][k], both row-major along k (k a multiple of 64, zero-padded).  D's layout puts four consecutive m
// of one n into a lane.  A workgroup computes BM x BN; k tiles of 64 go from HBM / L2 straight into LDS (buffer loads to LDS, 16 bytes a lane), two deep: the
// next tile is on its way while this one is multiplied.  A row of a tile is 128 bytes = all banks once, so the 16-byte pieces of row r are stored
// at piece ^ (r & 7): the 16 rows that a wave reads at a time then touch each bank equally.  The swizzle is applied to the address that a
// lane loads from, since the LDS side of such a load is lane after lane.
struct CeMat {
  const unsigned short* p;
  int64_t ld, plane;
};

template <int BM, int BN, int WM, int WN>
struct CeTile {
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // 1 KB loads per wave
  static constexpr int LDS = 2 * (BM + BN) * BK;                  // bf16 elements
  f32x4 acc[MT][NT];

  __device__ __forceinline__ void run(const CeMat& A, const CeMat& B, int m0, int M, int n0, int N, int k0, int k1, int pairs, unsigned short* lds) {
#if defined(__HIP_DEVICE_COMPILE__)  // the buffer resource's type is the device's alone
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int nk = (k1 - k0) / BK, total = nk > 0 ? nk * pairs : 0;
    // rows behind the last one read it again: what they give is never stored
    uint32_t va[LA], vb[LB];
    const int rl = lane >> 3, piece = (lane & 7) ^ rl;
#pragma unroll
    for (int i = 0; i < LA; ++i) va[i] = (uint32_t)min((i * WAVES + wave) * 8 + rl, M - 1 - m0) * (uint32_t)A.ld * 2u + piece * 16u;
#pragma unroll
    for (int i = 0; i < LB; ++i) vb[i] = (uint32_t)min((i * WAVES + wave) * 8 + rl, N - 1 - n0) * (uint32_t)B.ld * 2u + piece * 16u;
    const unsigned short* const a0 = A.p + (int64_t)m0 * A.ld;
    const unsigned short* const b0 = B.p + (int64_t)n0 * B.ld;

    auto stage = [&](int pr, int k, int buf) {
      const int pa = pairs == 1 ? 0 : CE_PAIRS_A >> (2 * pr) & 3, pb = pairs == 1 ? 0 : CE_PAIRS_B >> (2 * pr) & 3;
      const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(a0 + pa * A.plane), 0, 0xffffffff, 0x00020000);
      const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(b0 + pb * B.plane), 0, 0xffffffff, 0x00020000);
      unsigned short* const sa = lds + buf * (BM + BN) * BK;
      unsigned short* const sb = sa + BM * BK;
#pragma unroll
      for (int i = 0; i < LA; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(sa + (i * WAVES + wave) * 512), 16, va[i], k * 2, 0, 0);
#pragma unroll
      for (int i = 0; i < LB; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void*)(sb + (i * WAVES + wave) * 512), 16, vb[i], k * 2, 0, 0);
    };

    int pr = 0, k = k0;  // of the tile that is fetched next
    if (total > 0) stage(0, k0, 0);
    const int r = lane & 15, q = lane >> 4;
    for (int it = 0; it < total; ++it) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // this tile is there, and nobody reads the other buffer any more
      if (pairs > 1 && k == k0 && (pr == 3 || pr == 5)) {  // the first tile of a product that the ones so far are 2^-8 of
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] *= 0x1p-8f;
      }
      k += BK;
      if (k >= k1) { k = k0; ++pr; }
      if (it + 1 < total) stage(pr, k, (it + 1) & 1);
      const unsigned short* const sa = lds + (it & 1) * (BM + BN) * BK + (wm * MT * 16 + r) * BK;
      const unsigned short* const sb = lds + (it & 1) * (BM + BN) * BK + BM * BK + (wn * NT * 16 + r) * BK;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int at = ((kk * 4 + q) ^ (r & 7)) * 8;
        bf16x8 a[MT], b[NT];
#pragma unroll
        for (int i = 0; i < MT; ++i) a[i] = *reinterpret_cast<const bf16x8*>(sa + i * 16 * BK + at);
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = *reinterpret_cast<const bf16x8*>(sb + j * 16 * BK + at);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
      }
    }
    __syncthreads();
#endif
  }
};

// Workgroups go to the eight XCDs in turn: give each XCD a run of consecutive tiles, which share operands in its L2
__device__ __forceinline__ int ce_xcd(int b, int n) {
  const int per = n / 8, rest = n % 8, x = b % 8, i = b / 8;
  return x * per + (x < rest ? x : rest) + i;
}

template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void ce_stats_kernel(CeMat W, CeMat h, const int32_t* __restrict__ n, const int32_t* __restrict__ yc, int v0, int Vc, int K,
                                                                int pairs, int tiles_n, int part0, int parts, float2* __restrict__ part, float* __restrict__ at_y) {
  using G = CeTile<BM, BN, WM, WN>;
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int id = ce_xcd(blockIdx.x, gridDim.x);
  const int tm = id / tiles_n, m0 = tm * BM, n0 = id % tiles_n * BN, N = n[0];
  if (n0 >= N) return;
  G g;
  g.run(W, h, m0, Vc, n0, N, 0, K, pairs, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
  float2* const s = reinterpret_cast<float2*>(lds);  // [WM][BN]
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int cl = (wn * G::NT + j) * 16 + (lane & 15), t = n0 + cl;
    const int y = t < N ? yc[t] - v0 : -1;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < G::MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int v = m0 + (wm * G::MT + i) * 16 + 4 * q + k;
        if (v >= Vc) g.acc[i][j][k] = -INFINITY;
        else if (v == y) at_y[t] = g.acc[i][j][k];
        top = fmaxf(top, g.acc[i][j][k]);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < G::MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += __expf(g.acc[i][j][k] - base);
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (q == 0) s[wm * BN + cl] = make_float2(top, sum);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < BN; c += G::THREADS) {
    if (n0 + c >= N) continue;
    float2 v = s[c];
#pragma unroll
    for (int w = 1; w < WM; ++w) {
      const float2 u = s[w * BN + c];
      const float top = fmaxf(v.x, u.x), base = top == -INFINITY ? 0.f : top;
      v = make_float2(top, v.y * __expf(v.x - base) + u.y * __expf(u.x - base));
    }
    part[(int64_t)(n0 + c) * parts + part0 + tm] = v;
  }
}

// one wave per token that counts: joins the pieces' maxima and sums
__global__ __launch_bounds__(256) void ce_lse_kernel(const int32_t* __restrict__ n, const float2* __restrict__ part, int parts, const float* __restrict__ at_y,
                                                     const int32_t* __restrict__ yc, float* __restrict__ lse, float* __restrict__ loss) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (j >= n[0]) return;
  float top = -INFINITY;
  for (int c = lane; c < parts; c += 64) top = fmaxf(top, part[j * parts + c].x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int c = lane; c < parts; c += 64) {
    const float2 u = part[j * parts + c];
    sum += u.y * __expf(u.x - base);
  }
  sum = ceeg_wave_sum(sum);
  if (lane == 0) {
    const float l = base + logf(sum);
    lse[j] = l;
    loss[j] = yc[j] >= 0 ? l - at_y[j] : __uint_as_float(0x7fc00000u);  // a class outside [0, V) cannot raise an error from here: its loss is NaN
  }
}

// reduction 0: loss[t] for every token (0 where ignored); 1: mean over the tokens that count (0 where none does); 2: sum
__global__ __launch_bounds__(1024) void ce_loss_kernel(const int32_t* __restrict__ n, const float* __restrict__ rowloss, const int32_t* __restrict__ pos, int64_t T,
                                                       int reduction, float* __restrict__ loss) {
  if (reduction == 0) {
    const int64_t t = (int64_t)blockIdx.x * 1024 + threadIdx.x;
    if (t < T) loss[t] = pos[t] >= 0 ? rowloss[pos[t]] : 0.f;
    return;
  }
  __shared__ double s[16];
  double v = 0.0;
  for (int j = threadIdx.x; j < n[0]; j += 1024) v += (double)rowloss[j];
  v = ceeg_wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0;
    for (int k = 0; k < 16; ++k) v += s[k];
    loss[0] = (float)(reduction == 1 ? v / (n[0] > 0 ? n[0] : 1) : v);
  }
}

// scale[0] = s, r[j]: what comes back for token j is s r_j.  Mean and sum: r = 1, so that rounding r (p - [v = y]) to bf16 does not round the common factor too.
__global__ __launch_bounds__(1024) void ce_scale_kernel(const int32_t* __restrict__ n, const int32_t* __restrict__ rows, const int32_t* __restrict__ yc,
                                                        const float* __restrict__ g, int reduction, float* __restrict__ scale, float* __restrict__ r) {
  __shared__ float s[16];
  const int N = n[0];
  float top = 1.f;
  if (reduction == 0) {
    top = 0.f;
    for (int j = threadIdx.x; j < N; j += 1024) top = fmaxf(top, fabsf(g[rows[j]]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int k = 0; k < 16; ++k) top = fmaxf(top, s[k]);
  }
  for (int j = threadIdx.x; j < N; j += 1024) {
    float v = reduction == 0 ? (top > 0.f ? g[rows[j]] / top : g[rows[j]]) : 1.f;
    if (yc[j] < 0) v = __uint_as_float(0x7fc00000u);
    r[j] = v;
  }
  if (threadIdx.x == 0) scale[0] = reduction == 0 ? top : reduction == 1 ? g[0] / (float)(N > 0 ? N : 1) : g[0];
}

// dl of one piece of the vocabulary, [P][T][ldv] and [P][ldv][Tp]
template <int P, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void ce_dlogits_kernel(CeMat W, CeMat h, const int32_t* __restrict__ n, const int32_t* __restrict__ yc,
                                                                  const float* __restrict__ lse, const float* __restrict__ r, int v0, int Vc, int ldv, int64_t T, int64_t Tp,
                                                                  int K, int pairs, int tiles_n, unsigned short* __restrict__ dl, unsigned short* __restrict__ dlT) {
  using G = CeTile<BM, BN, WM, WN>;
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int id = ce_xcd(blockIdx.x, gridDim.x);
  const int m0 = id / tiles_n * BM, n0 = id % tiles_n * BN, N = n[0];
  if (n0 >= N) return;
  G g;
  g.run(W, h, m0, Vc, n0, N, 0, K, pairs, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
  const int Nz = (N + 63) & ~63;  // the transposed copy is summed over its tokens in steps of 64: zero behind the last
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int t = n0 + (wn * G::NT + j) * 16 + (lane & 15);
    const int y = t < N ? yc[t] - v0 : -1;
    const float l = t < N ? lse[t] : 0.f, rt = t < N ? r[t] : 0.f;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      const int v = m0 + (wm * G::MT + i) * 16 + 4 * q;
      if (v >= ldv) continue;
      unsigned short p[4][3];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x = 0.f;
        if (t < N && v + k < Vc) x = rt * (__expf(g.acc[i][j][k] - l) - (v + k == y ? 1.f : 0.f));
        if (P == 3) ce_split(x, p[k]); else p[k][0] = ceeg_f32_to_bf16(x);
      }
#pragma unroll
      for (int a = 0; a < P; ++a) {
        if (t < N) *reinterpret_cast<ushort4*>(dl + (a * T + t) * ldv + v) = make_ushort4(p[0][a], p[1][a], p[2][a], p[3][a]);
        if (t < Nz) {
#pragma unroll
          for (int k = 0; k < 4; ++k) dlT[((int64_t)a * ldv + v + k) * Tp + t] = p[k][a];
        }
      }
    }
  }
}

// dh += dl W of one piece: split over the vocabulary into slots that are joined at the end, [slots][T][H]
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void ce_dh_kernel(CeMat WT, CeMat dl, const int32_t* __restrict__ n, int H, int64_t T, int K, int k_slot, int pairs,
                                                             int tiles_m, int tiles, int add, float* __restrict__ slots) {
  using G = CeTile<BM, BN, WM, WN>;
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int id = ce_xcd(blockIdx.x, gridDim.x);
  const int slot = id / tiles, rest = id % tiles;
  const int m0 = rest % tiles_m * BM, n0 = rest / tiles_m * BN, N = n[0];
  if (n0 >= N) return;
  const int k0 = min(slot * k_slot, K), k1 = min(k0 + k_slot, K);
  G g;
  g.run(WT, dl, m0, H, n0, N, k0, k1, pairs, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int t = n0 + (wn * G::NT + j) * 16 + (lane & 15);
    if (t >= N) continue;
    float* const row = slots + (slot * T + t) * H;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      const int c = m0 + (wm * G::MT + i) * 16 + 4 * q;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < H) row[c + k] = add ? row[c + k] + g.acc[i][j][k] : g.acc[i][j][k];
    }
  }
}

// dW = s dl^T h of one piece
template <bool F32, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void ce_dw_kernel(CeMat hT, CeMat dlT, const int32_t* __restrict__ n, const float* __restrict__ scale, int H, int Vc, int pairs,
                                                             int tiles_m, void* __restrict__ dw) {
  using G = CeTile<BM, BN, WM, WN>;
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int id = ce_xcd(blockIdx.x, gridDim.x);
  const int m0 = id % tiles_m * BM, n0 = id / tiles_m * BN, K = (n[0] + 63) & ~63;
  G g;
  g.run(hT, dlT, m0, H, n0, Vc, 0, K, pairs, lds);
  const float s = scale[0];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int v = n0 + (wn * G::NT + j) * 16 + (lane & 15);
    if (v >= Vc) continue;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      const int c = m0 + (wm * G::MT + i) * 16 + 4 * q;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (c + k >= H) continue;
        // no token counts: the empty sum is zero whatever comes back
        const float x = K == 0 ? 0.f : s * g.acc[i][j][k];
        if (F32) static_cast<float*>(dw)[(int64_t)v * H + c + k] = x;
        else static_cast<unsigned short*>(dw)[(int64_t)v * H + c + k] = ceeg_f32_to_bf16(x);
      }
    }
  }
}

template <bool F32>
__global__ __launch_bounds__(256) void ce_dh_join_kernel(const float* __restrict__ part, int slots, const int32_t* __restrict__ pos, const float* __restrict__ scale, int64_t T,
                                                         int H, void* __restrict__ dh) {
  const int64_t t = blockIdx.x;
  const int j = pos[t];
  const float s = scale[0];
  for (int c = threadIdx.x; c < H; c += 256) {
    float x = 0.f;
    if (j >= 0) {
      for (int k = 0; k < slots; ++k) x += part[(k * T + j) * H + c];
      x *= s;
    }
    if (F32) static_cast<float*>(dh)[t * H + c] = x;
    else static_cast<unsigned short*>(dh)[t * H + c] = ceeg_f32_to_bf16(x);
  }
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int TB = 128;  // tile
inline int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

struct CePlan {
  int P, pairs;
  bool direct;           // W is read where it is
  int64_t Kp, Tp;        // padded H, padded T
  int64_t piece, ldv;    // columns of a piece of the vocabulary, padded
  int pieces, slots;
};

CePlan ce_plan(int64_t T, int64_t H, int64_t V, int dtype, bool backward) {
  CePlan c;
  c.P = dtype == CEEG_F32 ? 3 : 1;
  c.pairs = dtype == CEEG_F32 ? 6 : 1;
  c.direct = dtype == CEEG_BF16 && H % BK == 0;
  c.Kp = up(H, BK);
  c.Tp = up(T, BK);
  const int64_t column = c.P * ((backward ? 4 * c.Tp + 2 * H : 0) + (c.direct ? 0 : 2 * c.Kp));
  int64_t piece = V;
  if (column > 0 && piece > CE_CAP / column) piece = CE_CAP / column;
  if (piece > CE_MAX_PIECE) piece = CE_MAX_PIECE;
  if (piece < TB) piece = TB;
  c.pieces = (int)((V + piece - 1) / piece);
  c.piece = up((V + c.pieces - 1) / c.pieces, TB);
  c.pieces = (int)((V + c.piece - 1) / c.piece);
  c.ldv = up(c.piece < V ? c.piece : V, BK);
  // dh: few tiles (T H against V columns of sum), so the sum is cut until about two workgroups per compute unit are busy
  const int64_t tiles = ((T + TB - 1) / TB) * ((H + TB - 1) / TB);
  int64_t s = (512 + tiles - 1) / tiles;
  if (s > c.ldv / (4 * BK)) s = c.ldv / (4 * BK);
  if (s > 64) s = 64;
  c.slots = (int)(s < 1 ? 1 : s);
  return c;
}

bool ce_sizes_ok(int64_t T, int64_t H, int64_t V) { return T >= 1 && H >= 1 && V >= 1 && T <= (1 << 22) && H <= (1 << 15) && V <= (1 << 28); }

int ce_check(const void* h, int64_t ldh, const void* W, int64_t ldw, int64_t T, int64_t H, int64_t V, int dtype) {
  if (!h || !W || T < 1 || H < 1 || V < 1 || ldh < H || ldw < H) return CEEG_EINVAL;
  if (dtype != CEEG_F32 && dtype != CEEG_BF16) return CEEG_EUNSUPPORTED;
  if (!ce_sizes_ok(T, H, V) || ldw > (1 << 22)) return CEEG_EUNSUPPORTED;
  const size_t e = dtype == CEEG_F32 ? 4 : 2;
  if (!ceeg_aligned(h, e) || !ceeg_aligned(W, e)) return CEEG_EINVAL;
  if (dtype == CEEG_BF16 && H % BK == 0 && (ldw % 8 || !ceeg_aligned(W, 16))) return CEEG_EINVAL;
  return CEEG_OK;
}

size_t ce_fwd_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  const CePlan c = ce_plan(T, H, V, dtype, false);
  const size_t parts = (size_t)(V + TB - 1) / TB;
  return ceeg_ws_part((size_t)c.P * T * c.Kp, 2) + (c.direct ? 0 : ceeg_ws_part((size_t)c.P * c.piece * c.Kp, 2)) + ceeg_ws_part((size_t)T * parts, 8) +
         2 * ceeg_ws_part(T, 4);
}
size_t ce_bwd_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  const CePlan c = ce_plan(T, H, V, dtype, true);
  return ceeg_ws_part((size_t)c.P * T * c.Kp, 2) + ceeg_ws_part((size_t)c.P * H * c.Tp, 2) + (c.direct ? 0 : ceeg_ws_part((size_t)c.P * c.piece * c.Kp, 2)) +
         ceeg_ws_part((size_t)c.P * H * c.ldv, 2) + ceeg_ws_part((size_t)c.P * T * c.ldv, 2) + ceeg_ws_part((size_t)c.P * c.ldv * c.Tp, 2) +
         ceeg_ws_part((size_t)c.slots * T * H, 4) + ceeg_ws_part(1, 4) + ceeg_ws_part(T, 4);
}

void ce_pack(int dtype, const void* src, int64_t ld, const int32_t* rows, const int32_t* count, int64_t R, int64_t C, unsigned short* out, int64_t plane, int64_t Cp,
             unsigned short* outT, int64_t planeT, int64_t Rp, hipStream_t st) {
  const dim3 grid((unsigned)((R + 63) / 64), (unsigned)((C + 63) / 64));
  if (dtype == CEEG_F32) ce_pack_kernel<true><<<grid, 256, 0, st>>>(src, ld, rows, count, (int)R, (int)C, out, plane, (int)Cp, outT, planeT, Rp);
  else ce_pack_kernel<false><<<grid, 256, 0, st>>>(src, ld, rows, count, (int)R, (int)C, out, plane, (int)Cp, outT, planeT, Rp);
}
inline const void* ce_at(const void* p, int64_t n, int dtype) { return static_cast<const char*>(p) + n * (dtype == CEEG_F32 ? 4 : 2); }
}  // namespace

extern "C" size_t ceeg_linear_ce_fwd_ws_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  return ce_sizes_ok(T, H, V) ? ce_fwd_bytes(T, H, V, dtype) : 0;
}
extern "C" size_t ceeg_linear_ce_bwd_ws_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  return ce_sizes_ok(T, H, V) ? ce_bwd_bytes(T, H, V, dtype) : 0;
}

extern "C" int ceeg_linear_ce_fwd(const void* h, int64_t ldh, const void* W, int64_t ldw, const int64_t* y, int64_t T, int64_t H, int64_t V, int dtype, int64_t ignore_index,
                                  int reduction, float* loss, float* lse, int32_t* tokens, void* ws, size_t ws_bytes, void* stream) {
  const int rc = ce_check(h, ldh, W, ldw, T, H, V, dtype);
  if (rc) return rc;
  if (!y || !ceeg_aligned(y, 8) || !loss || !lse || !tokens || reduction < 0 || reduction > 2) return CEEG_EINVAL;
  if (!ws || !ceeg_aligned(ws, 256) || ws_bytes < ce_fwd_bytes(T, H, V, dtype)) return CEEG_EWORKSPACE;
  const CePlan c = ce_plan(T, H, V, dtype, false);
  const int parts = (int)((V + TB - 1) / TB);
  CeegWs w(ws, ws_bytes);
  unsigned short* hc = w.take<unsigned short>((size_t)c.P * T * c.Kp);
  unsigned short* wc = c.direct ? nullptr : w.take<unsigned short>((size_t)c.P * c.piece * c.Kp);
  float2* part = w.take<float2>((size_t)T * parts);
  float* at_y = w.take<float>(T);
  float* rowloss = w.take<float>(T);
  if (!w.ok) return CEEG_EWORKSPACE;
  int32_t *n = tokens, *rows = tokens + 1, *pos = rows + T, *yc = pos + T;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  ce_tokens_kernel<<<1, 1024, 0, st>>>(y, T, V, ignore_index, n, rows, pos, yc);
  CEEG_CHECK_LAUNCH();
  ce_pack(dtype, h, ldh, rows, n, T, H, hc, T * c.Kp, c.Kp, nullptr, 0, 0, st);
  CEEG_CHECK_LAUNCH();
  const int tiles_n = (int)((T + TB - 1) / TB);
  const CeMat Bm{hc, c.Kp, T * c.Kp};
  for (int p = 0; p < c.pieces; ++p) {
    const int64_t v0 = p * c.piece, Vc = V - v0 < c.piece ? V - v0 : c.piece;
    CeMat A{static_cast<const unsigned short*>(W) + v0 * ldw, ldw, 0};
    if (!c.direct) {
      ce_pack(dtype, ce_at(W, v0 * ldw, dtype), ldw, nullptr, nullptr, Vc, H, wc, c.piece * c.Kp, c.Kp, nullptr, 0, 0, st);
      CEEG_CHECK_LAUNCH();
      A = CeMat{wc, c.Kp, c.piece * c.Kp};
    }
    const int tiles_m = (int)((Vc + TB - 1) / TB);
    ce_stats_kernel<TB, TB, 2, 2><<<tiles_m * tiles_n, 256, 0, st>>>(A, Bm, n, yc, (int)v0, (int)Vc, (int)c.Kp, c.pairs, tiles_n, (int)(v0 / TB), parts, part, at_y);
    CEEG_CHECK_LAUNCH();
  }
  ce_lse_kernel<<<(unsigned)((T + 3) / 4), 256, 0, st>>>(n, part, parts, at_y, yc, lse, rowloss);
  CEEG_CHECK_LAUNCH();
  ce_loss_kernel<<<reduction == 0 ? (unsigned)((T + 1023) / 1024) : 1u, 1024, 0, st>>>(n, rowloss, pos, T, reduction, loss);
  CEEG_CHECK_LAUNCH();
  return CEEG_OK;
}

extern "C" int ceeg_linear_ce_bwd(const void* h, int64_t ldh, const void* W, int64_t ldw, int64_t T, int64_t H, int64_t V, int dtype, int reduction, const float* g,
                                  const float* lse, const int32_t* tokens, void* dh, void* dw, void* ws, size_t ws_bytes, void* stream) {
  const int rc = ce_check(h, ldh, W, ldw, T, H, V, dtype);
  if (rc) return rc;
  if (!g || !lse || !tokens || (!dh && !dw) || reduction < 0 || reduction > 2) return CEEG_EINVAL;
  if (!ws || !ceeg_aligned(ws, 256) || ws_bytes < ce_bwd_bytes(T, H, V, dtype)) return CEEG_EWORKSPACE;
  const CePlan c = ce_plan(T, H, V, dtype, true);
  CeegWs w(ws, ws_bytes);
  unsigned short* hc = w.take<unsigned short>((size_t)c.P * T * c.Kp);
  unsigned short* hT = w.take<unsigned short>((size_t)c.P * H * c.Tp);
  unsigned short* wc = c.direct ? nullptr : w.take<unsigned short>((size_t)c.P * c.piece * c.Kp);
  unsigned short* WT = w.take<unsigned short>((size_t)c.P * H * c.ldv);
  unsigned short* dl = w.take<unsigned short>((size_t)c.P * T * c.ldv);
  unsigned short* dlT = w.take<unsigned short>((size_t)c.P * c.ldv * c.Tp);
  float* slots = w.take<float>((size_t)c.slots * T * H);
  float* scale = w.take<float>(1);
  float* r = w.take<float>(T);
  if (!w.ok) return CEEG_EWORKSPACE;
  const int32_t *n = tokens, *rows = tokens + 1, *pos = rows + T, *yc = pos + T;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  ce_scale_kernel<<<1, 1024, 0, st>>>(n, rows, yc, g, reduction, scale, r);
  CEEG_CHECK_LAUNCH();
  ce_pack(dtype, h, ldh, rows, n, T, H, hc, T * c.Kp, c.Kp, hT, H * c.Tp, c.Tp, st);
  CEEG_CHECK_LAUNCH();
  const int tiles_t = (int)((T + TB - 1) / TB), tiles_h = (int)((H + TB - 1) / TB);
  for (int p = 0; p < c.pieces; ++p) {
    const int64_t v0 = p * c.piece, Vc = V - v0 < c.piece ? V - v0 : c.piece, ldv = up(Vc, BK);
    CeMat A{static_cast<const unsigned short*>(W) + v0 * ldw, ldw, 0};
    ce_pack(dtype, ce_at(W, v0 * ldw, dtype), ldw, nullptr, nullptr, Vc, H, wc, c.piece * c.Kp, c.Kp, WT, H * ldv, ldv, st);
    CEEG_CHECK_LAUNCH();
    if (!c.direct) A = CeMat{wc, c.Kp, c.piece * c.Kp};
    const int tiles_v = (int)((Vc + TB - 1) / TB);
    const CeMat Bm{hc, c.Kp, T * c.Kp};
    if (c.P == 3)
      ce_dlogits_kernel<3, TB, TB, 2, 2><<<tiles_v * tiles_t, 256, 0, st>>>(A, Bm, n, yc, lse, r, (int)v0, (int)Vc, (int)ldv, T, c.Tp, (int)c.Kp, c.pairs, tiles_t, dl, dlT);
    else
      ce_dlogits_kernel<1, TB, TB, 2, 2><<<tiles_v * tiles_t, 256, 0, st>>>(A, Bm, n, yc, lse, r, (int)v0, (int)Vc, (int)ldv, T, c.Tp, (int)c.Kp, c.pairs, tiles_t, dl, dlT);
    CEEG_CHECK_LAUNCH();
    if (dh) {
      const int k_slot = (int)up((ldv + c.slots - 1) / c.slots, BK);
      ce_dh_kernel<TB, TB, 2, 2><<<tiles_h * tiles_t * c.slots, 256, 0, st>>>(CeMat{WT, ldv, H * ldv}, CeMat{dl, ldv, T * ldv}, n, (int)H, T, (int)ldv, k_slot, c.pairs, tiles_h,
                                                                              tiles_h * tiles_t, p > 0, slots);
      CEEG_CHECK_LAUNCH();
    }
    if (dw) {
      const CeMat At{hT, c.Tp, H * c.Tp}, Bt{dlT, c.Tp, ldv * c.Tp};
      if (dtype == CEEG_F32)
        ce_dw_kernel<true, TB, TB, 2, 2><<<tiles_h * tiles_v, 256, 0, st>>>(At, Bt, n, scale, (int)H, (int)Vc, c.pairs, tiles_h, static_cast<float*>(dw) + v0 * H);
      else
        ce_dw_kernel<false, TB, TB, 2, 2><<<tiles_h * tiles_v, 256, 0, st>>>(At, Bt, n, scale, (int)H, (int)Vc, c.pairs, tiles_h, static_cast<unsigned short*>(dw) + v0 * H);
      CEEG_CHECK_LAUNCH();
    }
  }
  if (dh) {
    if (dtype == CEEG_F32) ce_dh_join_kernel<true><<<(unsigned)T, 256, 0, st>>>(slots, c.slots, pos, scale, T, (int)H, dh);
    else ce_dh_join_kernel<false><<<(unsigned)T, 256, 0, st>>>(slots, c.slots, pos, scale, T, (int)H, dh);
    CEEG_CHECK_LAUNCH();
  }
  return CEEG_OK;
}
