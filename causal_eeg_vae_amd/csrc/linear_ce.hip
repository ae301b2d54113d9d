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
// bf16 inputs: dl is rounded to bf16 before both gradient products (half a step, 2^-8 of a value, at most), because the instruction takes bf16 and three planes of it would be
// three products; the common factor s stays out of it.  A gradient is 5e-4 to 7e-4 of its rms off one from an fp32 dl at
// the sizes below, 2e-3 at small ones; its own rounding to bf16 is 1.1e-3 to 2.3e-3.  lse is one fp32 number: a probability of the backward is off by 2^-24 |lse| of itself.
// The vocabulary is taken in pieces; of a piece only dl is held.  A product whose operand runs across the summed axis (W in dh, h and dl in
// dW) reads it through the transposing LDS read, so nothing is ever stored transposed.  No float atomics: the pieces of a sum are added in a fixed order.
// Measured, bf16, 8192 tokens (7373 count) x 1024 x 131072: statistics 1.73 ms (1.14 PFLOP/s), and per half of the vocabulary dl 0.96 ms (1.03), dh 0.81 ms (1.21),
// dW 0.81 ms (1.23); 1.13 over all, the recomputed logits counted, 0.85 without.  fp32, 16384 x 256 x 4096: 197, 226, 188 and 166 us (1.05, 0.91, 1.10, 1.24 PFLOP/s of bf16
// products, a sixth of that in fp32).
#include <limits.h>
#include "ceeg_internal.h"

namespace {
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using i32x4 = __attribute__((ext_vector_type(4))) int;

constexpr int PAD = 64;                                  // rows and columns of the packed operands are padded to this with zeros
constexpr int64_t CE_CAP = (int64_t)1 << 30;             // bytes that a piece of the vocabulary may take, where 256 columns of it take less
constexpr int CE_SCAN = 4096;                           // tokens whose places a workgroup finds by itself
constexpr int64_t CE_MAX_PIECE = (int64_t)1 << 20;       // columns per piece: 32-bit offsets inside a tile
__host__ __device__ constexpr int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

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
// rows[j] = j-th token that counts, pos[t] = j or -1, yc[j] = its class (-1: outside [0, V)), n[0] = how many; `zeros`, where given, is cleared where a token does not.
struct CeTokens {
  const int64_t* y;
  int64_t T, V, ignore;
  int32_t *n, *rows, *pos, *yc;
  float* zeros;
};

// All of them by one workgroup; `write`: into memory; `places` (LDS): pos, for up to CE_SCAN tokens.  Returns how many count.  4096 tokens a turn: every wave counts in
// EACH stretches of 64 (loads and stores lane after lane), the 64 counts are summed up by one wave.
template <int THREADS>
__device__ __forceinline__ int ce_scan(const CeTokens& a, bool write, int32_t* places) {
  constexpr int WAVES = THREADS / 64, EACH = 64 / WAVES;
  __shared__ int s_sum[65];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int64_t t0 = 0; t0 < a.T; t0 += 4096) {
    int64_t v[EACH];
    uint64_t on[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int64_t t = t0 + k * THREADS + threadIdx.x;
      v[k] = a.ignore;
      if (t0 + k * THREADS < a.T && t < a.T) v[k] = a.y[t];
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      on[k] = __ballot(v[k] != a.ignore);
      if (lane == 0) s_sum[k * WAVES + wave] = __popcll(on[k]);
    }
    __syncthreads();
    if (wave == 0) {
      const int mine = s_sum[lane];
      int pre = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(pre, o, 64);
        if (lane >= o) pre += u;
      }
      s_sum[lane] = pre - mine;
      if (lane == 63) s_sum[64] = pre;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int64_t t = t0 + k * THREADS + threadIdx.x;
      if (t0 + k * THREADS >= a.T) break;
      const bool counts = on[k] >> lane & 1;
      const int j = base + s_sum[k * WAVES + wave] + __popcll(on[k] & ((1ull << lane) - 1));
      if (t >= a.T) continue;
      if (places) places[t] = counts ? j : -1;
      if (write) {
        a.pos[t] = counts ? j : -1;
        if (counts) {
          a.rows[j] = (int32_t)t;
          a.yc[j] = v[k] >= 0 && v[k] < a.V ? (int32_t)v[k] : -1;
        } else if (a.zeros) {
          a.zeros[t] = 0.f;
        }
      }
    }
    base += s_sum[64];
    __syncthreads();
  }
  if (write && threadIdx.x == 0) a.n[0] = base;
  return base;
}

__global__ __launch_bounds__(1024) void ce_tokens_kernel(CeTokens a) { ce_scan<1024>(a, true, nullptr); }

// ------------------------------------------------------------------------------------------------ planes
// Where element (r, c) of a blocked matrix of C columns is: blocks of 16 rows x 32 columns, each one piece of 1 KB, so that a tile's loads are whole cache lines whichever way the tile
// lies.  Rows of 32 columns from a row-major matrix are half lines, twice the requests: 3 to 5 % of the products' time.
__host__ __device__ __forceinline__ int64_t ce_place(int64_t r, int c, int64_t C) { return ((r >> 4) * (C >> 5) + (c >> 5)) * 512 + (r & 15) * 32 + (c & 31); }

// eight columns c.. of a row of C at `src` (NULL: zeros) -> the planes at out
template <bool F32>
__device__ __forceinline__ void ce_pack8(const void* src, int c, int C, unsigned short* out, int64_t plane) {
  float x[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = 0.f;
  if (src) {
    if (F32) {
      const float* q = static_cast<const float*>(src) + c;
      if (c + 8 <= C && (reinterpret_cast<uintptr_t>(q) & 15) == 0) {
        const float4 u = reinterpret_cast<const float4*>(q)[0], v = reinterpret_cast<const float4*>(q)[1];
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = c + k < C ? q[k] : 0.f;
      }
    } else {
      const unsigned short* q = static_cast<const unsigned short*>(src) + c;
      if (c + 8 <= C && (reinterpret_cast<uintptr_t>(q) & 15) == 0) {
        *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(q);
        return;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = c + k < C ? ceeg_bf16_to_f32(q[k]) : 0.f;
    }
  }
  unsigned short p[8][3];
#pragma unroll
  for (int k = 0; k < 8; ++k) ce_split(x[k], p[k]);
#pragma unroll
  for (int a = 0; a < (F32 ? 3 : 1); ++a)
    *reinterpret_cast<uint4*>(out + a * plane) =
        make_uint4(p[0][a] | (uint32_t)p[1][a] << 16, p[2][a] | (uint32_t)p[3][a] << 16, p[4][a] | (uint32_t)p[5][a] << 16, p[6][a] | (uint32_t)p[7][a] << 16);
}

// Row-major [R, C] -> planes [P][*][Cp] (blocked where there are three), columns C..Cp zero; `zeros`: the rows behind the last, up to the next multiple of PAD, zero too (a sum over the rows runs over them).
template <bool F32>
__global__ __launch_bounds__(256) void ce_pack_kernel(const void* __restrict__ src, int64_t ld, int64_t R, int C, int Cp, int zeros, unsigned short* __restrict__ out, int64_t plane) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = Cp / 8;
  const int64_t r = id / per;
  const int c = (int)(id % per) * 8;
  if (r >= (zeros ? up(R, PAD) : R)) return;
  ce_pack8<F32>(r < R ? static_cast<const char*>(src) + r * ld * (F32 ? 4 : 2) : nullptr, c, C, out + (F32 ? ce_place(r, c, Cp) : r * Cp + c), plane);
}

// The hidden states of the tokens that count, packed and blocked; `each` tokens per workgroup, the last workgroup adds the zero rows.  SCAN: up to CE_SCAN tokens, whose places every
// workgroup finds for itself (a few KB from L2) - one launch instead of two; otherwise ce_tokens_kernel has found them.  V = H = 256 forward: 64 tokens 16.3 us, 17.4
// with two launches; 4096 20.4 and 20.3; 16384 44.7 and 37.4.
template <bool F32, int SCAN>
__device__ __forceinline__ void ce_prepare(const CeTokens& a, const void* __restrict__ h, int64_t ld, int H, int Kp, int each, int block, int blocks, unsigned short* __restrict__ out, int64_t plane) {
  __shared__ int32_t s_pos[SCAN ? SCAN : 1];
  int n;
  if (SCAN) {
    n = ce_scan<256>(a, block == 0, s_pos);
    __syncthreads();
  } else {
    n = a.n[0];
  }
  const int per = Kp / 8;
  const int64_t t0 = (int64_t)block * each;
  for (int i = threadIdx.x; i < each * per; i += 256) {
    const int64_t t = t0 + i / per;
    if (t >= a.T) break;
    const int j = SCAN ? s_pos[t] : a.pos[t], c = i % per * 8;
    if (j >= 0) ce_pack8<F32>(static_cast<const char*>(h) + t * ld * (F32 ? 4 : 2), c, H, out + ce_place(j, c, Kp), plane);
  }
  if (block == blocks - 1) {
    const int rows = (int)up(n, PAD) - n;
    for (int i = threadIdx.x; i < rows * per; i += 256) ce_pack8<F32>(nullptr, i % per * 8, H, out + ce_place(n + i / per, i % per * 8, Kp), plane);
  }
}
template <bool F32, bool SCAN>
__global__ __launch_bounds__(256) void ce_prepare_kernel(CeTokens a, const void* __restrict__ h, int64_t ld, int H, int Kp, int each, unsigned short* __restrict__ out, int64_t plane) {
  ce_prepare<F32, SCAN ? CE_SCAN : 0>(a, h, ld, H, Kp, each, blockIdx.x, gridDim.x, out, plane);
}

// ------------------------------------------------------------------------------------------------ products
// D[n][m] = sum_k A[m][k] B[n][k].  The 16 x 16 result layout puts four consecutive m of one n into a lane, so D's rows are stored in pieces of four.
// An operand lies along k ("row r holds r's k", 16-byte LDS reads) or across it ("row k holds all r", transposing LDS reads, which hand a
// lane four consecutive k of its r).  A workgroup computes BM x BN; tiles of BK elements of k go from HBM / L2 straight into LDS (buffer loads to LDS, 16 bytes a
// lane), ST deep: while one is multiplied the next ones are on their way, with one barrier a tile.
// Bank conflicts: the LDS side of such a load is lane after lane, so the swizzle is applied to the address that a lane loads from.  Along k a row of the tile is
// 64 bytes and its 16-byte pieces are stored at piece ^ (r / 2 mod 4): eight rows read together touch all banks once.  Across k the
// 32-byte pieces (one 16 x 16 block) of row k are stored at piece ^ (k mod 4 + 4 (k / 8 mod 2)): the eight rows that half a wave reads then lie in eight
// different pieces.
// Three planes (fp32): of every k tile all planes are in LDS and the six products run from there; the planes' powers of two keep three accumulators,
// joined at the end, small ones first.
#if defined(__HIP_DEVICE_COMPILE__)
// 16 bytes a lane from a buffer's base + v into LDS, lane after lane.  Written out because the compiler, which knows that such a load writes LDS, would
// wait for all of them before every transposing read; run() waits for exactly those it needs.  It has no output register.  m0, the
// place in LDS, is an input that the compiler sets (and computes in place); it takes a wait state to be read.
__device__ __forceinline__ void ce_to_lds(i32x4 rsrc, uint32_t v, unsigned short* to) {
  const uint32_t at = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)to);
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(at), "v"(v), "s"(rsrc) : "memory");
}
#endif

template <int N> struct Int { static constexpr int value = N; };
struct CeMat {
  const unsigned short* p;
  int64_t ld, plane;
  int r_end;                   // rows r there are: what lies behind is not read (the buffer's range check) and what it gives is never stored
  const unsigned short* tail;  // across k: the last rows k, from k_tail on, zero-padded to PAD, lie here where the matrix itself is not padded
  int k_tail;
};

template <int PL, int BM, int BN, int WM, int WN, int ST, bool AHEAD, bool TA, bool TB>
struct CeTile {
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int BK = 32;  // one matrix instruction deep
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static constexpr int LA = BM * BK / 512 / WAVES, LB = BN * BK / 512 / WAVES;  // 1 KB loads per wave, tile and plane
  static constexpr int PLANE = (BM + BN) * BK, STAGE = PL * PLANE;              // bf16 elements of LDS
  static constexpr int LDS = ST * STAGE;
  static_assert(LA > 0 && LB > 0 && LA * WAVES * 512 == BM * BK && LB * WAVES * 512 == BN * BK, "whole loads");
  static_assert(LDS * 2 <= 160 * 1024, "LDS");
  // B is always a matrix made here, and blocked; A is W, which in bf16 lies as the caller has it, or (both across k) the hidden states
  static constexpr bool BLOCKED_A = PL == 3 || (TA && TB);
  // A row-major along k, in the largest tile: two k tiles of it at a time, 128 bytes a row, for the same reason as the blocks' (8192 x 1024 x 131072 7.00 -> 6.91 ms,
  // 5000 x 768 x 50257 forward 279 -> 271 us).
  static constexpr bool PAIRS = !BLOCKED_A && !TA && BM == 256;
  f32x4 acc[MT][NT];

  // Load i of a wave fetches 64 pieces of 16 bytes of the tile: rows `row(lane) + hop(i)`; a hop changes no bit of a row that the swizzle looks at, so that
  // a lane's offset is the same for all loads.
  template <bool T, int BR>
  static __device__ __forceinline__ int hop(int i) {
    return !T ? i * WAVES * 16 : BR == 256 ? i * 4 : i * 16;
  }
  template <bool T, int BR>
  static __device__ __forceinline__ int row0(int wave) {
    return !T ? wave * 16 : BR == 256 ? (wave & 1) * 2 + (wave >> 1) * 8 : wave * (512 / BR);  // 256: eight waves
  }
  template <bool T, int BR, bool BLOCKED>
  static __device__ __forceinline__ uint32_t offset(const CeMat& x, int wave, int lane) {
    if (T) {
      constexpr int CPR = BR / 8;  // pieces per row k
      const int row = row0<T, BR>(wave) + lane / CPR, slot = lane % CPR, g = ((row & 3) | (row >> 3 & 1) << 2) & (BR / 16 - 1);
      const uint32_t piece = (uint32_t)(((slot >> 1) ^ g) << 1 | (slot & 1));
      if (BLOCKED) return (uint32_t)(lane / CPR) * 64u + (piece >> 2) * 1024u + (piece & 3u) * 16u;
      return (uint32_t)(lane / CPR) * (uint32_t)x.ld * 2u + piece * 16u;
    }
    const int row = lane >> 2;
    return (uint32_t)row * (BLOCKED ? 64u : (uint32_t)x.ld * 2u) + (uint32_t)((lane & 3) ^ (row >> 1 & 3)) * 16u;
  }
  // bytes that may be read from the tile's first element on: to the end of its last row
  template <bool T>
  static __device__ __forceinline__ int64_t range(const CeMat& x, int r0) {
    return T ? ((BK - 1) * x.ld + x.r_end - r0) * 2 : ((int64_t)(x.r_end - 1 - r0) * x.ld + BK) * 2;
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // k0 < k1, both multiples of PAD: at least two tiles, and an even number of them
  __device__ __forceinline__ void run(const CeMat& A, const CeMat& B, int m0, int n0, int k0, int k1, unsigned short* lds) {
#if defined(__HIP_DEVICE_COMPILE__)  // the buffer resource's type is the device's alone
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, l15 = lane & 15, q = lane >> 4;
    clear();
    f32x4 low[PL == 3 ? 2 : 1][MT][NT];
    if constexpr (PL == 3) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) low[0][i][j] = low[1][i][j] = acc[i][j];
    }
    const int total = (k1 - k0) / BK;
    const uint32_t va = offset<TA, BM, BLOCKED_A>(A, wave, lane), vb = offset<TB, BN, true>(B, wave, lane);
    const int64_t na = range<TA>(A, m0);

    auto to_lds = [&](const unsigned short* p, int64_t left, uint32_t v, unsigned short* to) {
      const uint64_t base = reinterpret_cast<uint64_t>(p);
      const i32x4 rs = {(int)(uint32_t)base, (int)(uint32_t)(base >> 32), left < 0 ? 0 : left > 0x7fffffff ? 0x7fffffff : (int)left, 0x00020000};
      ce_to_lds(rs, v, to);
    };
    auto fetch = [&](auto t, auto br, auto n, auto blocked, const CeMat& x, int r0, int k, int64_t bytes, uint32_t v, unsigned short* to) {
      constexpr bool T = decltype(t)::value != 0;
      constexpr int BR = decltype(br)::value;
      const unsigned short* p = x.p + (T ? (int64_t)k * x.ld + r0 : (int64_t)r0 * x.ld + k);
      if (!decltype(blocked)::value && T && k >= x.k_tail) p = x.tail + (int64_t)(k - x.k_tail) * x.ld + r0;
#pragma unroll
      for (int a = 0; a < PL; ++a) {
#pragma unroll
        for (int i = 0; i < n.value; ++i) {
          const int r = row0<T, BR>(wave) + hop<T, BR>(i);
          unsigned short* const at = to + a * PLANE + r * (T ? BR : BK);
          const int64_t strip = x.ld >> 5;  // blocks of a row of blocks
          if (!decltype(blocked)::value) to_lds(p + a * x.plane + r * x.ld, bytes - r * x.ld * 2, v, at);
          else if (T) to_lds(x.p + a * x.plane + (((k + r) >> 4) * strip + (r0 >> 5)) * 512 + (r & 15) * 32, (strip - (r0 >> 5)) * 1024 - (r & 15) * 64, v, at);  // to the end of the row of blocks
          else to_lds(x.p + a * x.plane + (((r0 + r) >> 4) * strip + (k >> 5)) * 512, ((r0 + r) & ~15) < x.r_end ? 1024 : 0, v, at);
        }
      }
    };
    // PAIRS: [2][BM][2 BK] of A, then [4][BN][BK] of B.  A row is 128 bytes, piece p of 16 at p ^ (r / 2 mod 8): 16 rows read together touch all banks once.
    unsigned short* const lds_b = lds + 2 * BM * 2 * BK;
    const uint32_t vp = (uint32_t)(lane >> 3) * (uint32_t)A.ld * 2u + (uint32_t)((lane & 7) ^ ((wave & 1) << 2 | lane >> 4)) * 16u;
    auto stage_a = [&](int pair) {
      const unsigned short* const p = A.p + (int64_t)m0 * A.ld + k0 + pair * 2 * BK;
#pragma unroll
      for (int i = 0; i < 2 * LA; ++i) {
        const int r = wave * 8 + i * WAVES * 8;
        to_lds(p + r * A.ld, na + 2 * BK - r * A.ld * 2, vp, lds + (pair & 1) * BM * 2 * BK + r * 2 * BK);
      }
    };
    auto stage_b = [&](int it) { fetch(Int<TB>{}, Int<BN>{}, Int<LB>{}, Int<1>{}, B, n0, k0 + it * BK, 0, vb, lds_b + (it & 3) * BN * BK); };
    auto stage = [&](int it) {
      const int k = k0 + it * BK;
      unsigned short* const to = lds + it % ST * STAGE;
      fetch(Int<TA>{}, Int<BM>{}, Int<LA>{}, Int<BLOCKED_A>{}, A, m0, k, na, va, to);
      fetch(Int<TB>{}, Int<BN>{}, Int<LB>{}, Int<1>{}, B, n0, k, 0, vb, to + BM * BK);
    };
    // waits until tile `it` is there for every wave; `ahead`: how many tiles behind it have been asked for.  Every wave has then read all that it read before.
    auto arrive_when = [&](bool more, auto loads) {
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(loads.value) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last tiles: nothing is asked for behind them
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    auto arrive = [&](int it, auto ahead) { arrive_when(it + ahead.value < total, Int<ahead.value * PL * (LA + LB)>{}); };
    const int g = (l15 >> 2) | (q & 1) << 2, at = (q ^ (l15 >> 1 & 3)) * 8, row = 8 * q + (l15 >> 2);
    auto read_a = [&](int it, int p, int i) {
      if (PAIRS) return *reinterpret_cast<const bf16x8*>(lds + (it >> 1 & 1) * BM * 2 * BK + ((wm * MT + i) * 16 + l15) * 2 * BK + (((it & 1) * 4 + q) ^ l15 >> 1) * 8);
      return read<TA, BM>(lds + it % ST * STAGE + p * PLANE, wm * MT + i, l15, at, row, g);
    };
    auto read_b = [&](int it, int p, int j) {
      return read<TB, BN>(PAIRS ? lds_b + (it & 3) * BN * BK : lds + it % ST * STAGE + p * PLANE + BM * BK, wn * NT + j, l15, at, row, g);
    };

    if constexpr (AHEAD) {
      // The next tile's fragments are read while this one's are multiplied, so that after a barrier no wave waits for LDS before it can go on.
      static_assert(!PAIRS || (ST == 4 && PL == 1), "two pairs, four tiles");
      if (PAIRS) {
        stage_a(0);
        stage_b(0);
        stage_b(1);
        if (total > 2) {
          stage_a(1);
          stage_b(2);
          stage_b(3);
        }
      } else {
#pragma unroll
        for (int s = 0; s < ST; ++s)
          if (s < total) stage(s);
      }
      struct Frag {
        bf16x8 a[MT], b[NT];
      };
      auto load = [&](Frag& f, int it) {
#pragma unroll
        for (int j = 0; j < NT; ++j) f.b[j] = read_b(it, 0, j);
#pragma unroll
        for (int i = 0; i < MT; ++i) f.a[i] = read_a(it, 0, i);
      };
      auto mul = [&](const Frag& f) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.a[i], f.b[j], acc[i][j], 0, 0, 0);
      };
      Frag f0, f1;
      // PAIRS: the order is A of tiles 0 and 1, B0, B1, A of 2 and 3, B2, B3, B4, A of 4 and 5, B5, B6, ...
      if (PAIRS) arrive_when(total > 2, Int<2 * LA + 3 * LB>{});
      else arrive(0, Int<ST - 1>{});
      load(f0, 0);
      auto step = [&](int it, auto odd, const Frag& now, Frag& next) {
        if (PAIRS) {
          arrive_when(it + 3 < total, Int<odd.value ? 2 * LB : 2 * LA + 2 * LB>{});
          if (odd.value && it + 3 < total) stage_a((it + 3) >> 1);
          if (it + 4 < total) stage_b(it + 4);
        } else {
          arrive(it + 1, Int<ST - 2>{});
          if (it + ST < total) stage(it + ST);
        }
        load(next, it + 1);
        mul(now);
        constexpr int READS = MT * (TA ? 2 : 1) + NT * (TB ? 2 : 1), EACH = MT * NT / READS;
#pragma unroll
        for (int i = 0; i < READS; ++i) {  // a read between every few products
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        }
      };
      for (int it = 0; it + 2 < total; it += 2) {
        step(it, Int<0>{}, f0, f1);
        step(it + 1, Int<1>{}, f1, f0);
      }
      step(total - 2, Int<0>{}, f0, f1);
      mul(f1);
    } else {
#pragma unroll
      for (int s = 0; s < ST - 1; ++s)
        if (s < total) stage(s);
      for (int it = 0; it < total; ++it) {
        arrive(it, Int<ST - 2>{});
        if (it + ST - 1 < total) stage(it + ST - 1);
        bf16x8 a[PL][MT], b[PL][NT];
#pragma unroll
        for (int p = 0; p < PL; ++p) {
#pragma unroll
          for (int j = 0; j < NT; ++j) b[p][j] = read_b(it, p, j);
#pragma unroll
          for (int i = 0; i < MT; ++i) a[p][i] = read_a(it, p, i);
        }
        auto mul = [&](f32x4 (&to)[MT][NT], int pa, int pb) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) to[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[pa][i], b[pb][j], to[i][j], 0, 0, 0);
        };
        if constexpr (PL == 3) {
          mul(low[1], 2, 0); mul(low[1], 0, 2); mul(low[1], 1, 1);
          mul(low[0], 1, 0); mul(low[0], 0, 1);
        }
        mul(acc, 0, 0);
      }
    }
    if constexpr (PL == 3) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          // An infinite factor lies in its first plane alone and meets the other's lower planes, zeros and other signs among them: where the first planes'
          // sum is not finite, it is the sum.  (Selected by value: elements of a vector written under conditions of their own came out of the
          // compiler as copies of the first.)
          const f32x4 x = acc[i][j], y = x + (low[0][i][j] + low[1][i][j] * 0x1p-8f) * 0x1p-8f;
          const auto pick = [](float a, float b) { return fabsf(a) <= 3.402823466e38f ? b : a; };
          acc[i][j] = f32x4{pick(x[0], y[0]), pick(x[1], y[1]), pick(x[2], y[2]), pick(x[3], y[3])};
        }
    }
    __syncthreads();
#endif
  }

#if defined(__HIP_DEVICE_COMPILE__)
  template <bool T, int BR>
  static __device__ __forceinline__ bf16x8 read(const unsigned short* s, int block, int l15, int at, int row, int g) {
    if (!T) return *reinterpret_cast<const bf16x8*>(s + (block * 16 + l15) * BK + at);
    using s16x4 = __attribute__((ext_vector_type(4))) short;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const unsigned short* const p = s + row * BR + ((block ^ (g & (BR / 16 - 1))) * 16 + (l15 & 3) * 4);
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * BR));  // rows 4 further swizzle the same
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
#endif
};

// The tile shapes.  256 x 256 on eight waves reads LDS least per product and fills the chip from 256 tiles up (one workgroup per compute unit); 128 x 128 halves what is lost on
// smaller grids; 64 x 64 spreads the smallest, which are bound by latency, and keeps more tiles on their way.
template <int PL, bool TA, bool TB> struct CeBig { using Tile = CeTile<1, 256, 256, 2, 4, 4, true, TA, TB>; };
template <int PL, bool TA, bool TB> struct CeMid { using Tile = CeTile<1, 128, 128, 2, 2, 4, true, TA, TB>; };
template <bool TA, bool TB> struct CeMid<3, TA, TB> { using Tile = CeTile<3, 128, 64, 2, 2, 2, false, TA, TB>; };
template <int PL, bool TA, bool TB> struct CeSmall { using Tile = CeTile<1, 64, 64, 2, 2, 8, true, TA, TB>; };
template <bool TA, bool TB> struct CeSmall<3, TA, TB> { using Tile = CeTile<3, 64, 64, 2, 2, 3, false, TA, TB>; };

// exp(x - base).  bf16: one fused multiply-add in front of the instruction, whose rounding of base * log2(e) is worth 2^-24 |base| of the result; fp32: the difference first.
template <int PL>
__device__ __forceinline__ float ce_exp(float x, float base) {
  constexpr float LOG2E = 1.44269504088896341f;
  return __builtin_amdgcn_exp2f(PL == 1 ? __fmaf_rn(x, LOG2E, -base * LOG2E) : (x - base) * LOG2E);
}
// bf16: a base whose product with log2(e) may overflow takes fp32's form, in its own lane: the other tokens' numbers do not depend on it
__device__ __forceinline__ bool ce_far(float base) { return fabsf(base) > 0x1p126f; }
template <int PL, bool FAR>
__device__ __forceinline__ float ce_exp_of(float x, float base) { return FAR && ce_far(base) ? ce_exp<3>(x, base) : ce_exp<PL>(x, base); }

// four consecutive values of a row of H (left: how many of them there are), in the output's type
template <bool F32>
__device__ __forceinline__ void ce_store4(void* to, int64_t at, int left, int H, float a, float b, float c, float d) {
  const float x[4] = {a, b, c, d};
  if ((H & 3) == 0) {
    if (F32) *reinterpret_cast<float4*>(static_cast<float*>(to) + at) = make_float4(a, b, c, d);
    else *reinterpret_cast<ushort4*>(static_cast<unsigned short*>(to) + at) = make_ushort4(ceeg_f32_to_bf16(a), ceeg_f32_to_bf16(b), ceeg_f32_to_bf16(c), ceeg_f32_to_bf16(d));
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= left) continue;
    if (F32) static_cast<float*>(to)[at + k] = x[k];
    else static_cast<unsigned short*>(to)[at + k] = ceeg_f32_to_bf16(x[k]);
  }
}

// Edge along n of the tile with this edge along m
__host__ __device__ __forceinline__ int ce_n(int planes, int edge) { return planes == 3 ? 64 : edge; }
__host__ __device__ __forceinline__ int64_t ce_tiles(int planes, int edge, int64_t m, int64_t n) {
  const int en = ce_n(planes, edge);
  return ((m + edge - 1) / edge) * ((n + en - 1) / en);
}

// Workgroups go to the eight XCDs in turn: each XCD gets a run of consecutive tiles (-1: none left for this workgroup) ...
__device__ __forceinline__ int ce_xcd(int b, int n) {
  const int per = n / 8, rest = n % 8, x = b % 8, i = b / 8;
  return i < per + (x < rest) ? x * per + (x < rest ? x : rest) + i : -1;
}
// ... which are taken in bands of six along n, so that the 32 tiles which the XCD's compute units work on at a time share six by five operands in its L2
__device__ __forceinline__ void ce_band(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int W = 6;
  const int band = id / (W * tiles_m), in = id - band * W * tiles_m, w = min(W, tiles_n - band * W);
  tm = in / w;
  tn = band * W + in - tm * w;
}

template <class G, int PL, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(G::THREADS, 1) void ce_stats_kernel(CeMat W, CeMat h, const int32_t* __restrict__ n, const int32_t* __restrict__ yc, int v0, int K, int part0,
                                                              int parts, float2* __restrict__ part, float* __restrict__ at_y) {
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int N = n[0], Vc = W.r_end, tiles_m = (Vc + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
  const int id = ce_xcd(blockIdx.x, tiles_m * tiles_n);
  if (id < 0) return;
  int tm, tn;
  ce_band(id, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  h.r_end = N;
  G g;
  g.run(W, h, m0, n0, 0, K, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
  float2* const s = reinterpret_cast<float2*>(lds);  // [WM][BN]
  const int vb = m0 + wm * G::MT * 16;
  // About 7 instructions a logit are a fifth of the product's time at H = 1024: the mask of the last tile and the search for the tokens' own classes
  // run only where a wave has some.
  if (vb + G::MT * 16 > Vc) {
#pragma unroll
    for (int i = 0; i < G::MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (vb + i * 16 + 4 * q + k >= Vc) {
#pragma unroll
          for (int j = 0; j < G::NT; ++j) g.acc[i][j][k] = -INFINITY;
        }
  }
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int cl = (wn * G::NT + j) * 16 + (lane & 15), t = n0 + cl;
    const int y = t < N ? yc[t] - v0 - vb : -1;
    if (__any(y >= 0 && y < G::MT * 16)) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i * 16 + 4 * q + k == y) at_y[t] = g.acc[i][j][k];
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) top = fmaxf(top, fmaxf(fmaxf(g.acc[i][j][0], g.acc[i][j][1]), fmaxf(g.acc[i][j][2], g.acc[i][j][3])));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    const auto add = [&](auto far) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += ce_exp_of<PL, far.value>(g.acc[i][j][k], base);
    };
    if (PL == 1 && __any(ce_far(base))) add(Int<1>{});
    else add(Int<0>{});
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

// A wave joins the maxima and sums c, c + step, ... (c: its first, plus the lane) that the tiles left of a token: one pass, eight loads a lane in flight
__device__ __forceinline__ float2 ce_join(const float2* __restrict__ part, int c, int step, int parts) {
  float top = -INFINITY, sum = 0.f;
  for (int64_t c0 = c; c0 < parts; c0 += 8 * (int64_t)step) {
    float2 u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = c0 + (int64_t)step * k < parts ? part[c0 + (int64_t)step * k] : make_float2(-INFINITY, 0.f);
    float t = top;
#pragma unroll
    for (int k = 0; k < 8; ++k) t = fmaxf(t, u[k].x);
    const float base = t == -INFINITY ? 0.f : t;
    sum *= __expf(top - base);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += u[k].y * __expf(u[k].x - base);
    top = t;
  }
  float t = top;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
  const float base = t == -INFINITY ? 0.f : t;
  return make_float2(t, ceeg_wave_sum(sum * __expf(top - base)));
}
__device__ __forceinline__ float ce_lse(float2 v) { return (v.x == -INFINITY ? 0.f : v.x) + logf(v.y); }
// a class outside [0, V) cannot raise an error from here: its loss is NaN
__device__ __forceinline__ float ce_row_loss(float lse, const float* __restrict__ at_y, const int32_t* __restrict__ yc, int64_t j) {
  return yc[j] >= 0 ? lse - at_y[j] : __uint_as_float(0x7fc00000u);
}

// loss of token j to rowloss[j] (rows NULL) or to rowloss[rows[j]]
__global__ __launch_bounds__(256) void ce_lse_kernel(const int32_t* __restrict__ n, const float2* __restrict__ part, int parts, const float* __restrict__ at_y,
                                                     const int32_t* __restrict__ yc, const int32_t* __restrict__ rows, float* __restrict__ lse, float* __restrict__ rowloss) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (j >= n[0]) return;
  const float l = ce_lse(ce_join(part + j * parts, lane, 64, parts));
  if (lane == 0) {
    lse[j] = l;
    rowloss[rows ? rows[j] : j] = ce_row_loss(l, at_y, yc, j);
  }
}

// Mean over the tokens that count (0 where none does) or sum, one workgroup.  A launch of its own also for few tokens: one workgroup that finds their lse on the way takes
// longer than a wave each (32 tokens of 256 classes 19.0 us instead of 16.7 for the whole loss, 1 of 50257 21.3 instead of 18.4).
__global__ __launch_bounds__(1024) void ce_loss_kernel(const int32_t* __restrict__ n, const float* __restrict__ rowloss, int reduction, float* __restrict__ loss) {
  __shared__ double s[16];
  const int N = n[0], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double v = 0.0;
  for (int j = threadIdx.x; j < N; j += 1024) v += (double)rowloss[j];
  v = ceeg_wave_sum_d(v);
  if (lane == 0) s[wave] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0;
    for (int k = 0; k < 16; ++k) v += s[k];
    loss[0] = (float)(reduction == 1 ? v / (N > 0 ? N : 1) : v);
  }
}

// ------------------------------------------------------------------------------------------------ few tokens
// The statistics of up to R tokens against W read once as it is (no planes, no padding, fp32 multiply-adds): bound by W's bytes.  16 lanes take four rows of W, a wave sixteen, a
// workgroup FEW of them; the hidden rows are in LDS in fp32, read once for the four rows; two pieces of 16 bytes of each row are on their way.  A last workgroup
// does what ce_prepare_kernel does meanwhile.  One token x 768 x 50257: bf16 15.6 us (4.9 TB/s, W
// in the 256 MB cache from the call before); with the join in fp32 30 us, in bf16 19.0, and 21.6 where the weights of twelve calls take turns and W comes from memory.
constexpr int CE_FEW = 64;             // classes of a workgroup
constexpr int CE_FEW_TOKENS = 8;
constexpr int CE_FEW_LDS = 48 * 1024;  // bytes of hidden rows

template <bool F32, int R, bool WIDE>
__global__ __launch_bounds__(256, R == 1 ? 4 : R == 2 ? 3 : 2) void ce_few_kernel(CeTokens a, const void* __restrict__ h, int64_t ldh, const void* __restrict__ W, int64_t ldw, int H, int Kp, int parts,
                                                        float2* __restrict__ part, float* __restrict__ at_y, unsigned short* __restrict__ packed, int64_t plane) {
  constexpr int VEC = F32 ? 4 : 8, U = 4;
  extern __shared__ __align__(16) float s_h[];  // [R][Hv]
  __shared__ float2 s_wave[4][R];
  const int blocks = (int)gridDim.x - 1;
  if ((int)blockIdx.x == blocks) {
    ce_prepare<F32, CE_FEW_TOKENS>(a, h, ldh, H, Kp, CE_FEW_TOKENS, 0, 1, packed, plane);
    return;
  }
  const int Hv = (int)up(H, 32 * VEC), passes = Hv / (16 * VEC), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, l = lane & 15;
  const int64_t y = lane < a.T ? a.y[lane] : a.ignore;  // T <= R
  // 16 bytes of each of the four rows, zeros behind H.  WIDE: all of W in pieces of 16 bytes on such addresses
  const auto load = [&](uint4 (&w)[U], int b, int pass) {
    const int c = (pass * 16 + l) * VEC;
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = make_uint4(0u, 0u, 0u, 0u);
    if (c >= H || b >= parts) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int64_t v = (int64_t)b * CE_FEW + wave * 16 + group * U + u;
      if (v >= a.V) v = a.V - 1;  // what it gives is not looked at
      const char* const q = static_cast<const char*>(W) + (v * ldw + c) * (F32 ? 4 : 2);
      if (WIDE) {
        w[u] = *reinterpret_cast<const uint4*>(q);
      } else {
        uint32_t x[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          if (c + k >= H) continue;
          if (F32) x[k % 4] = reinterpret_cast<const uint32_t*>(q)[k];
          else x[k / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(q)[k] << (16 * (k & 1));
        }
        w[u] = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
  };
  uint4 w0[U], w1[U];  // two passes on their way
  load(w0, blockIdx.x, 0);
  load(w1, blockIdx.x, 1);
  uint64_t left = __ballot(y != a.ignore);
  const int N = __popcll(left);
  int cls[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int t = left ? __ffsll((unsigned long long)left) - 1 : 0;
    left &= left - 1;
    const int64_t own = __shfl(y, t, 64);
    cls[r] = r < N && own >= 0 && own < a.V ? (int)own : -1;
    for (int c = threadIdx.x; c < Hv; c += 256) {
      float x = 0.f;
      if (r < N && c < H) x = F32 ? static_cast<const float*>(h)[t * ldh + c] : ceeg_bf16_to_f32(static_cast<const unsigned short*>(h)[t * ldh + c]);
      s_h[r * Hv + c] = x;
    }
  }
  __syncthreads();
  for (int b = blockIdx.x; b < parts; b += blocks) {
    float acc[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) acc[u][r] = 0.f;
    const auto step = [&](uint4 (&w)[U], int pass) {  // multiplies a pass and asks for the one after the next
      float f[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t x[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int k = 0; k < VEC; ++k) f[u][k] = __uint_as_float(F32 ? x[k % 4] : k & 1 ? x[k / 2] & 0xffff0000u : x[k / 2] << 16);
      }
      const bool more = pass + 2 < passes;
      load(w, more ? b : b + blocks, more ? pass + 2 : pass + 2 - passes);
      const float* const x = s_h + (pass * 16 + l) * VEC;
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int k = 0; k < VEC; k += 4) {
          const float4 z = *reinterpret_cast<const float4*>(x + r * Hv + k);
#pragma unroll
          for (int u = 0; u < U; ++u)
            acc[u][r] = __fmaf_rn(f[u][k + 3], z.w, __fmaf_rn(f[u][k + 2], z.z, __fmaf_rn(f[u][k + 1], z.y, __fmaf_rn(f[u][k], z.x, acc[u][r]))));
        }
      }
    };
    for (int pass = 0; pass < passes; pass += 2) {
      step(w0, pass);
      step(w1, pass + 1);
    }
    const int64_t v0 = (int64_t)b * CE_FEW + wave * 16 + group * U;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) acc[u][r] += __shfl_xor(acc[u][r], o, 64);
        if (v0 + u >= a.V) acc[u][r] = -INFINITY;
        else if (l == 0 && cls[r] == v0 + u) at_y[r] = acc[u][r];
        top = fmaxf(top, acc[u][r]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) sum += ce_exp_of<F32 ? 3 : 1, !F32>(acc[u][r], base);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (lane == 0) s_wave[wave][r] = make_float2(top, sum);
    }
    __syncthreads();
    if ((int)threadIdx.x < N) {
      float2 v = s_wave[0][threadIdx.x];
      for (int k = 1; k < 4; ++k) {
        const float2 o = s_wave[k][threadIdx.x];
        const float top = fmaxf(v.x, o.x), base = top == -INFINITY ? 0.f : top;
        v = make_float2(top, v.y * __expf(v.x - base) + o.y * __expf(o.x - base));
      }
      part[(int64_t)threadIdx.x * parts + b] = v;
    }
    __syncthreads();
  }
}

// lse and loss of up to R tokens by one workgroup, 16 / R waves a token
template <int R>
__global__ __launch_bounds__(1024) void ce_few_loss_kernel(const int32_t* __restrict__ n, const float2* __restrict__ part, int parts, const float* __restrict__ at_y,
                                                           const int32_t* __restrict__ yc, const int32_t* __restrict__ rows, int reduction, float* __restrict__ lse, float* __restrict__ loss) {
  constexpr int EACH = 16 / R;
  __shared__ float2 s[16];
  const int N = n[0], lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = wave / EACH;
  float2 v = make_float2(-INFINITY, 0.f);
  if (mine < N) v = ce_join(part + (int64_t)mine * parts, wave % EACH * 64 + lane, EACH * 64, parts);
  if (lane == 0) s[wave] = v;
  __syncthreads();
  if (wave != 0) return;
  double d = 0.0;
  if (lane < N) {
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < EACH; ++k) top = fmaxf(top, s[lane * EACH + k].x);
    const float base = top == -INFINITY ? 0.f : top;
    for (int k = 0; k < EACH; ++k) sum += s[lane * EACH + k].y * __expf(s[lane * EACH + k].x - base);
    const float z = ce_lse(make_float2(top, sum)), x = ce_row_loss(z, at_y, yc, lane);
    lse[lane] = z;
    if (reduction == 0) loss[rows[lane]] = x;
    d = (double)x;
  }
  if (reduction == 0) return;
  d = ceeg_wave_sum_d(d);
  if (lane == 0) loss[0] = (float)(reduction == 1 ? d / (N > 0 ? N : 1) : d);
}

// What comes back for token j is s r_j.  Mean and sum: r = 1, so that rounding r (p - [v = y]) to bf16 does not round the common factor too.
struct CeScale {
  const float* g;
  int reduction;
  const float *top, *r;  // no reduction: s = the largest finite |g|, r_j = g_j / s; what is not finite is its token's own r and leaves the others' alone
  __device__ __forceinline__ float s(int N) const { return reduction == 0 ? top[0] : reduction == 1 ? g[0] / (float)(N > 0 ? N : 1) : g[0]; }
  __device__ __forceinline__ float row(int j, int y) const { return y < 0 ? __uint_as_float(0x7fc00000u) : reduction == 0 ? r[j] : 1.f; }
};
__global__ __launch_bounds__(1024) void ce_scale_kernel(const int32_t* __restrict__ n, const int32_t* __restrict__ rows, const float* __restrict__ g, float* __restrict__ scale,
                                                        float* __restrict__ r) {
  __shared__ float s[16];
  const int N = n[0];
  float top = 0.f;
  for (int j = threadIdx.x; j < N; j += 1024) {
    const float x = fabsf(g[rows[j]]);
    if (x <= 3.402823466e38f) top = fmaxf(top, x);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int k = 0; k < 16; ++k) top = fmaxf(top, s[k]);
  for (int j = threadIdx.x; j < N; j += 1024) r[j] = top > 0.f ? g[rows[j]] / top : g[rows[j]];
  if (threadIdx.x == 0) scale[0] = top;
}

// dl of one piece of the vocabulary, [P][T][ldv], blocked; columns behind the piece and the rows up to the next multiple of PAD are zero
template <class G, int PL, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(G::THREADS, 1) void ce_dlogits_kernel(CeMat W, CeMat h, const int32_t* __restrict__ n, const int32_t* __restrict__ yc, const float* __restrict__ lse,
                                                                CeScale scale, int v0, int ldv, int64_t plane, int K, unsigned short* __restrict__ dl) {
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int N = n[0], Vc = W.r_end, tiles_m = (Vc + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
  const int id = ce_xcd(blockIdx.x, tiles_m * tiles_n);
  if (id < 0) return;
  int tm, tn;
  ce_band(id, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  h.r_end = N;
  G g;
  g.run(W, h, m0, n0, 0, K, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
  const int Nz = (int)up(N, PAD), vb = m0 + wm * G::MT * 16;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int t = n0 + (wn * G::NT + j) * 16 + (lane & 15);
    const int class_t = t < N ? yc[t] : -1, y = class_t - v0 - vb;
    const float l = t < N ? lse[t] : 0.f, rt = t < N ? scale.row(t, class_t) : 0.f;
    const auto set = [&](auto far) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) g.acc[i][j][k] = rt * ce_exp_of<PL, far.value>(g.acc[i][j][k], l);
    };
    if (PL == 1 && __any(ce_far(l))) set(Int<1>{});
    else set(Int<0>{});
    if (__any(y >= 0 && y < G::MT * 16)) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i * 16 + 4 * q + k == y) g.acc[i][j][k] -= rt;
    }
    if (vb + G::MT * 16 > Vc || n0 + BN > N) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t >= N || vb + i * 16 + 4 * q + k >= Vc) g.acc[i][j][k] = 0.f;  // whatever was multiplied there
    }
    // through LDS (the tiles are done with), so that blocks leave in whole lines: token by token, its 16-byte pieces at piece ^ (token mod 16)
    const int tl = (wn * G::NT + j) * 16 + (lane & 15);
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      const int vl = (wm * G::MT + i) * 16 + 4 * q;
      f32x4 x = g.acc[i][j];
#pragma unroll
      for (int a = 0; a < PL; ++a) {
        const uint2 p = make_uint2(ceeg_f32_to_bf16x2(x[0], x[1]), ceeg_f32_to_bf16x2(x[2], x[3]));
        *reinterpret_cast<uint2*>(lds + a * BN * BM + tl * BM + (((vl >> 3) ^ (tl & (BM / 8 - 1) & 15)) * 8 + (vl & 4))) = p;
        if (a + 1 < PL) {  // what the plane leaves, 2^8 times
          x[0] = (x[0] - __uint_as_float(p.x << 16)) * 256.f;
          x[1] = (x[1] - __uint_as_float(p.x & 0xffff0000u)) * 256.f;
          x[2] = (x[2] - __uint_as_float(p.y << 16)) * 256.f;
          x[3] = (x[3] - __uint_as_float(p.y & 0xffff0000u)) * 256.f;
        }
      }
    }
  }
  __syncthreads();
  constexpr int PER = BM / 8;
  static_assert(PL * BN * BM <= G::LDS && BN * PER % G::THREADS == 0, "the tile fits");
#pragma unroll
  for (int a = 0; a < PL; ++a) {
#pragma unroll
    for (int c = 0; c < BN * PER / G::THREADS; ++c) {
      // a wave writes one block: 16 tokens x 32 columns
      const int block = (c * G::THREADS + threadIdx.x) >> 6, l = threadIdx.x & 63, tl = block / (BM / 32) * 16 + (l >> 2), piece = block % (BM / 32) * 4 + (l & 3);
      const int t = n0 + tl, v = m0 + piece * 8;
      if (t < Nz && v < ldv)
        *reinterpret_cast<uint4*>(dl + a * plane + ce_place(t, v, ldv)) = *reinterpret_cast<const uint4*>(lds + a * BN * BM + tl * BM + (piece ^ (tl & (PER - 1) & 15)) * 8);
    }
  }
}

// Into how many stretches a sum of k elements is cut for a grid of `tiles`, so that the compute units hold as many workgroups as their LDS allows (`want`), each with
// 256 elements at least.  dh: few tiles (tokens x H) against a long sum over the vocabulary; its tokens are counted on the device, and fewer of them mean more stretches.
struct CeCut {
  int want;        // 0: `most` is the number
  int most;
  int64_t room;    // rows of all slots together that there is memory for
};
__host__ __device__ __forceinline__ int ce_slots(const CeCut& c, int64_t tiles, int64_t rows, int64_t k) {
  if (c.want == 0) return c.most;
  int64_t s = c.want / (tiles > 0 ? tiles : 1);
  if (s > k / 256) s = k / 256;
  if (s > c.room / (rows > 0 ? rows : 1)) s = c.room / (rows > 0 ? rows : 1);
  if (s > 64) s = 64;
  return (int)(s < 1 ? 1 : s);
}

// D of a product into fp32 slots [slots][rows][H], each holding a stretch of the sum (k_slot elements): dh += dl W (rows: tokens, A = W, B = dl) or dW = dl^T h (rows:
// classes, A = h, B = dl).  A slot keeps its sum over the pieces (`add`).
template <class G, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(G::THREADS, 1) void ce_slots_kernel(CeMat A, CeMat B, const int32_t* __restrict__ n, int by_tokens, int H, int64_t rows, int K, int k_all, CeCut cut, int add,
                                                              float* __restrict__ out) {
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int N = n[0], end = by_tokens ? N : (int)rows;
  const int tiles_m = (H + BM - 1) / BM, tiles = tiles_m * ((end + BN - 1) / BN), slots = ce_slots(cut, tiles, end, k_all), id = ce_xcd(blockIdx.x, tiles * slots);
  if (id < 0) return;
  const int slot = id / tiles, rest = id - slot * tiles;
  const int m0 = rest % tiles_m * BM, n0 = rest / tiles_m * BN;
  if (by_tokens) {   // the rows are tokens
    B.r_end = N;
  } else {           // the sum is over tokens
    K = (int)up(N, PAD);
  }
  const int k_slot = (int)up((K + slots - 1) / slots, PAD), k0 = min(slot * k_slot, K), k1 = min(k0 + k_slot, K);
  G g;
  if (k0 < k1) {
    g.run(A, B, m0, n0, k0, k1, lds);
  } else {
    if (add) return;
    g.clear();
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int r = n0 + (wn * G::NT + j) * 16 + (lane & 15);
    if (r >= end) continue;
    float* const to = out + ((int64_t)slot * end + r) * H;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      const int c = m0 + (wm * G::MT + i) * 16 + 4 * q;
      if ((H & 3) == 0) {
        if (c < H) {
          float4* const f = reinterpret_cast<float4*>(to + c);
          float4 x = make_float4(g.acc[i][j][0], g.acc[i][j][1], g.acc[i][j][2], g.acc[i][j][3]);
          if (add) { const float4 y = *f; x = make_float4(y.x + x.x, y.y + x.y, y.z + x.z, y.w + x.w); }
          *f = x;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < H) to[c + k] = add ? to[c + k] + g.acc[i][j][k] : g.acc[i][j][k];
      }
    }
  }
}

// dW = s dl^T h of one piece, the whole sum in one workgroup
template <class G, bool F32, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(G::THREADS, 1) void ce_dw_kernel(CeMat h, CeMat dl, const int32_t* __restrict__ n, CeScale scale, int H, int Vc,
                                                           void* __restrict__ dw) {
  __shared__ __align__(16) unsigned short lds[G::LDS];
  const int tiles_m = (H + BM - 1) / BM, id = ce_xcd(blockIdx.x, gridDim.x);
  const int m0 = id % tiles_m * BM, n0 = id / tiles_m * BN, K = (int)up(n[0], PAD);
  G g;
  if (K > 0) g.run(h, dl, m0, n0, 0, K, lds);
  else g.clear();
  const float s = K == 0 ? 0.f : scale.s(n[0]);  // no token counts: the empty sum is zero whatever comes back
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int v = n0 + (wn * G::NT + j) * 16 + (lane & 15);
    if (v >= Vc) continue;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      const int c = m0 + (wm * G::MT + i) * 16 + 4 * q;
      if (c >= H) continue;
      ce_store4<F32>(dw, (int64_t)v * H + c, H - c, H, s * g.acc[i][j][0], s * g.acc[i][j][1], s * g.acc[i][j][2], s * g.acc[i][j][3]);
    }
  }
}

// the slots of dW joined
template <bool F32>
__global__ __launch_bounds__(256) void ce_dw_join_kernel(const float* __restrict__ part, int slots, const int32_t* __restrict__ n, CeScale scale, int64_t count,
                                                         void* __restrict__ dw) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  float x = 0.f;
  for (int k = 0; k < slots; ++k) x += part[k * count + i];
  x = n[0] == 0 ? 0.f : x * scale.s(n[0]);
  if (F32) static_cast<float*>(dw)[i] = x;
  else static_cast<unsigned short*>(dw)[i] = ceeg_f32_to_bf16(x);
}

// the slots of dh joined, four columns a thread, eight slots in flight; rows of tokens that do not count are zero
template <bool F32>
__global__ __launch_bounds__(256) void ce_dh_join_kernel(const float* __restrict__ part, int planes, int edge, int k_all, CeCut cut, const int32_t* __restrict__ n, const int32_t* __restrict__ pos,
                                                         CeScale scale, int64_t T, int H, void* __restrict__ dh) {
  const int per = (H + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, t = id / per;
  if (t >= T) return;
  const int N = n[0], j = pos[t], c = (int)(id - t * per) * 4;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (j >= 0) {
    const int slots = ce_slots(cut, ce_tiles(planes, edge, H, N), N, k_all);
    const float* const from = part + (int64_t)j * H + c;
    for (int k0 = 0; k0 < slots; k0 += 8) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float* const f = from + (int64_t)(k0 + k) * N * H;
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k0 + k >= slots) continue;
        if ((H & 3) == 0) v[k] = *reinterpret_cast<const float4*>(f);
        else v[k] = make_float4(f[0], c + 1 < H ? f[1] : 0.f, c + 2 < H ? f[2] : 0.f, c + 3 < H ? f[3] : 0.f);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) { x[0] += v[k].x; x[1] += v[k].y; x[2] += v[k].z; x[3] += v[k].w; }
    }
    const float s = scale.s(N);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] *= s;
  }
  ce_store4<F32>(dh, t * H + c, H - c, H, x[0], x[1], x[2], x[3]);
}

// ------------------------------------------------------------------------------------------------ host side
// Tile edge for a grid of rows x columns (x the ways its sum may be cut): the largest that gives (nearly) every compute unit a workgroup.  Forward, H = 512, 256 tiles of
// that edge: 256 x 256 32.6 us, 128 x 128 39.1 (T = 1024, V = 16384); 128 x 128 23.0 us, 64 x 64 25.3 (V = 4096).  With 128 tiles of it: 256 x 256
// 31.1 us, 128 x 128 27.2 (V = 8192); 128 x 128 20.2 us, 64 x 64 18.0 (H = 256, V = 2048).
int ce_edge(int planes, int64_t rows, int64_t cols, int64_t cuts) {
  const auto tiles = [&](int e) { return ce_tiles(planes, e, rows, cols); };
  if (planes == 1 && tiles(256) * cuts >= 200) return 256;
  if (tiles(128) * cuts >= 200) return 128;
  return 64;
}

// workgroups that the compute units hold at once
int ce_want(int edge) { return edge == 256 ? 256 : 512; }

struct CePlan {
  int P;
  bool direct;           // W is read where it is
  int64_t Kp, Tp;        // padded H, padded T
  int64_t piece, ldv;    // columns of a piece of the vocabulary, padded
  int pieces;
  int e_logits, e_dh, e_dw;         // tile edges
  CeCut dh_cut;                     // stretches that the sums are cut into
  int dw_slots;
  int few;                          // tokens that ce_few_kernel takes (a power of two), 0: the tiles
};

// Up to eight tokens in fp32, two in bf16: the tiles' time hardly depends on how few there are, as they first make planes of W (fp32) or pad it (bf16 of an H that is no multiple
// of 64).  768 x 50257: fp32 1 token 30 us, tiles 134; 8 tokens 48 and 139; bf16 1 token 19.0 and 28.5, 4 tokens 28.6 and 29.2, 8 tokens 41 and 30.
size_t ce_few_lds(int few, int64_t H, int dtype) { return (size_t)few * up(H, dtype == CEEG_F32 ? 128 : 256) * 4; }
int ce_few(int64_t T, int64_t H, int dtype) {
  if (T > (dtype == CEEG_F32 ? CE_FEW_TOKENS : 2)) return 0;
  const int r = T > 4 ? 8 : T > 2 ? 4 : (int)T;
  return ce_few_lds(r, H, dtype) <= CE_FEW_LDS ? r : 0;
}

CePlan ce_plan(int64_t T, int64_t H, int64_t V, int dtype, bool backward) {
  CePlan c;
  c.P = dtype == CEEG_F32 ? 3 : 1;
  c.direct = dtype == CEEG_BF16 && H % PAD == 0;
  c.Kp = up(H, PAD);
  c.Tp = up(T, PAD);
  const int64_t column = c.P * ((backward ? 2 * c.Tp : 0) + (c.direct ? 0 : 2 * c.Kp));
  int64_t piece = V;
  if (column > 0 && piece > CE_CAP / column) piece = CE_CAP / column;
  if (piece > CE_MAX_PIECE) piece = CE_MAX_PIECE;
  if (piece < 256) piece = 256;
  c.pieces = (int)((V + piece - 1) / piece);
  c.piece = up((V + c.pieces - 1) / c.pieces, 256);
  c.pieces = (int)((V + c.piece - 1) / c.piece);
  c.ldv = up(c.piece < V ? c.piece : V, PAD);
  const int64_t cols = c.piece < V ? c.piece : V;
  c.e_logits = ce_edge(c.P, cols, T, 1);
  c.few = backward ? 0 : ce_few(T, H, dtype);
  if (c.few) c.e_logits = CE_FEW;
  const auto tiles = [&](int64_t m, int64_t n, int e) { return ce_tiles(c.P, e, m, n); };
  c.e_dh = ce_edge(c.P, H, T, c.ldv / 1024 + 1);
  c.dh_cut = CeCut{ce_want(c.e_dh), 0, INT64_MAX};
  c.dh_cut.room = T * ce_slots(c.dh_cut, tiles(H, T, c.e_dh), T, c.ldv);
  c.e_dw = ce_edge(c.P, H, cols, T / 1024 + 1);
  // a sum over few tokens is short, so that a last round of large tiles that leaves compute units idle weighs more than their better rate (1152 x 768 x 50257:
  // 591 tiles of 256 in 3 rounds 131 us, 2358 of 128 in 5 half rounds 115 us)
  const auto fill = [&](int64_t n, int64_t at_once) { return (double)n / (double)up(n, at_once); };
  if (c.e_dw == 256 && T <= 2048 && fill(tiles(H, cols, 128), 512) > 1.15 * fill(tiles(H, cols, 256), 256)) c.e_dw = 128;
  c.dw_slots = tiles(H, cols, c.e_dw) >= 200 ? 1 : ce_slots(CeCut{ce_want(c.e_dw), 0, INT64_MAX}, tiles(H, cols, c.e_dw), 1, T);
  return c;
}

bool ce_sizes_ok(int64_t T, int64_t H, int64_t V) { return T >= 1 && H >= 1 && V >= 1 && T <= (1 << 22) && H <= (1 << 15) && V <= (1 << 28); }

int ce_check(const void* h, int64_t ldh, const void* W, int64_t ldw, int64_t T, int64_t H, int64_t V, int dtype) {
  if (!h || !W || T < 1 || H < 1 || V < 1 || ldh < H || ldw < H) return CEEG_EINVAL;
  if (dtype != CEEG_F32 && dtype != CEEG_BF16) return CEEG_EUNSUPPORTED;
  if (!ce_sizes_ok(T, H, V) || ldw > (1 << 22)) return CEEG_EUNSUPPORTED;
  const size_t e = dtype == CEEG_F32 ? 4 : 2;
  if (!ceeg_aligned(h, e) || !ceeg_aligned(W, e)) return CEEG_EINVAL;
  if (dtype == CEEG_BF16 && H % PAD == 0 && (ldw != H || !ceeg_aligned(W, 16))) return CEEG_EINVAL;
  return CEEG_OK;
}

size_t ce_packed_bytes(const CePlan& c) { return ceeg_ws_part((size_t)c.P * c.Tp * c.Kp, 2); }
size_t ce_fwd_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  const CePlan c = ce_plan(T, H, V, dtype, false);
  const size_t parts = (size_t)(V + c.e_logits - 1) / c.e_logits;
  return (c.direct || c.few ? 0 : ceeg_ws_part((size_t)c.P * c.piece * c.Kp, 2)) + ceeg_ws_part((size_t)T * parts, 8) + 2 * ceeg_ws_part(T, 4);
}
size_t ce_bwd_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  const CePlan c = ce_plan(T, H, V, dtype, true);
  return (c.direct ? ceeg_ws_part((size_t)PAD * c.Kp, 2) : ceeg_ws_part((size_t)c.P * c.piece * c.Kp, 2)) + ceeg_ws_part((size_t)c.P * c.Tp * c.ldv, 2) +
         ceeg_ws_part((size_t)c.dh_cut.room * H, 4) + (c.dw_slots > 1 ? ceeg_ws_part((size_t)c.dw_slots * c.piece * H, 4) : 0) + ceeg_ws_part(1, 4) + ceeg_ws_part(T, 4);
}

void ce_pack(int dtype, const void* src, int64_t ld, int64_t R, int64_t C, int64_t Cp, bool zeros, unsigned short* out, int64_t plane, hipStream_t st) {
  const unsigned grid = (unsigned)(((zeros ? up(R, PAD) : R) * (Cp / 8) + 255) / 256);
  if (dtype == CEEG_F32) ce_pack_kernel<true><<<grid, 256, 0, st>>>(src, ld, R, (int)C, (int)Cp, zeros, out, plane);
  else ce_pack_kernel<false><<<grid, 256, 0, st>>>(src, ld, R, (int)C, (int)Cp, zeros, out, plane);
}
inline const void* ce_at(const void* p, int64_t n, int dtype) { return static_cast<const char*>(p) + n * (dtype == CEEG_F32 ? 4 : 2); }

// CALL with (planes, edges along m and n, waves along each, tile type) of the edge chosen
#define CE_TILES(PLANES, EDGE, TA, TB, CALL)                                         \
  do {                                                                               \
    if ((PLANES) == 3) {                                                             \
      if ((EDGE) == 128) { CALL(3, 128, 64, 2, 2, (CeMid<3, TA, TB>::Tile)); }       \
      else { CALL(3, 64, 64, 2, 2, (CeSmall<3, TA, TB>::Tile)); }                    \
    } else {                                                                         \
      if ((EDGE) == 256) { CALL(1, 256, 256, 2, 4, (CeBig<1, TA, TB>::Tile)); }      \
      else if ((EDGE) == 128) { CALL(1, 128, 128, 2, 2, (CeMid<1, TA, TB>::Tile)); } \
      else { CALL(1, 64, 64, 2, 2, (CeSmall<1, TA, TB>::Tile)); }                    \
    }                                                                                \
  } while (0)
template <class> struct CeArg;
template <class X> struct CeArg<void(X)> { using type = X; };
#define CE_TILE_OF(T) typename CeArg<void T>::type
}  // namespace

extern "C" size_t ceeg_linear_ce_fwd_ws_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  return ce_sizes_ok(T, H, V) ? ce_fwd_bytes(T, H, V, dtype) : 0;
}
extern "C" size_t ceeg_linear_ce_bwd_ws_bytes(int64_t T, int64_t H, int64_t V, int dtype) {
  return ce_sizes_ok(T, H, V) ? ce_bwd_bytes(T, H, V, dtype) : 0;
}

extern "C" size_t ceeg_linear_ce_packed_bytes(int64_t T, int64_t H, int dtype) {
  return ce_sizes_ok(T, H, 1) ? ce_packed_bytes(ce_plan(T, H, 1, dtype, false)) : 0;
}

extern "C" int ceeg_linear_ce_fwd(const void* h, int64_t ldh, const void* W, int64_t ldw, const int64_t* y, int64_t T, int64_t H, int64_t V, int dtype, int64_t ignore_index,
                                  int reduction, float* loss, float* lse, int32_t* tokens, void* packed, void* ws, size_t ws_bytes, void* stream) {
  const int rc = ce_check(h, ldh, W, ldw, T, H, V, dtype);
  if (rc) return rc;
  if (!y || !ceeg_aligned(y, 8) || !loss || !lse || !tokens || reduction < 0 || reduction > 2) return CEEG_EINVAL;
  if (!packed || !ceeg_aligned(packed, 256)) return CEEG_EINVAL;
  if (!ws || !ceeg_aligned(ws, 256) || ws_bytes < ce_fwd_bytes(T, H, V, dtype)) return CEEG_EWORKSPACE;
  const CePlan c = ce_plan(T, H, V, dtype, false);
  const int parts = (int)((V + c.e_logits - 1) / c.e_logits);
  CeegWs w(ws, ws_bytes);
  unsigned short* const hc = static_cast<unsigned short*>(packed);
  unsigned short* wc = c.direct || c.few ? nullptr : w.take<unsigned short>((size_t)c.P * c.piece * c.Kp);
  float2* part = w.take<float2>((size_t)T * parts);
  float* at_y = w.take<float>(T);
  float* rowloss = w.take<float>(T);
  if (!w.ok) return CEEG_EWORKSPACE;
  int32_t *n = tokens, *rows = tokens + 1, *pos = rows + T, *yc = pos + T;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const CeTokens tk{y, T, V, ignore_index, n, rows, pos, yc, reduction == 0 ? loss : nullptr};
  if (c.few) {
    const size_t lds = ce_few_lds(c.few, H, dtype);
    const bool wide = ceeg_aligned(W, 16) && (dtype == CEEG_F32 ? (H | ldw) % 4 == 0 : (H | ldw) % 8 == 0);
    const int resident = 256 * (c.few == 1 ? 4 : c.few == 2 ? 3 : 2);
    const unsigned grid = (unsigned)(parts < resident ? parts : resident) + 1;  // what is resident at once, and the one that prepares
#define CE_CALL(F32, R)                                                                                                                                                 \
  do {                                                                                                                                                                  \
    if (wide) ce_few_kernel<F32, R, true><<<grid, 256, lds, st>>>(tk, h, ldh, W, ldw, (int)H, (int)c.Kp, parts, part, at_y, hc, c.Tp * c.Kp);                        \
    else ce_few_kernel<F32, R, false><<<grid, 256, lds, st>>>(tk, h, ldh, W, ldw, (int)H, (int)c.Kp, parts, part, at_y, hc, c.Tp * c.Kp);                            \
    CEEG_CHECK_LAUNCH();                                                                                                                                                \
    ce_few_loss_kernel<R><<<1, 1024, 0, st>>>(n, part, parts, at_y, yc, rows, reduction, lse, loss);                                                                    \
  } while (0)
    if (dtype == CEEG_F32) {
      if (c.few == 1) CE_CALL(true, 1);
      else if (c.few == 2) CE_CALL(true, 2);
      else if (c.few == 4) CE_CALL(true, 4);
      else CE_CALL(true, 8);
    } else {
      if (c.few == 1) CE_CALL(false, 1);
      else CE_CALL(false, 2);
    }
#undef CE_CALL
    CEEG_CHECK_LAUNCH();
    return CEEG_OK;
  }
  const bool scan = T <= CE_SCAN;
  if (!scan) {
    ce_tokens_kernel<<<1, 1024, 0, st>>>(tk);
    CEEG_CHECK_LAUNCH();
  }
  const int each = c.Kp / 8 >= 128 ? 8 : (int)(1024 / (c.Kp / 8));  // about 1024 pieces of 16 bytes a workgroup
  const unsigned grid = (unsigned)((T + each - 1) / each);
  if (dtype == CEEG_F32) {
    if (scan) ce_prepare_kernel<true, true><<<grid, 256, 0, st>>>(tk, h, ldh, (int)H, (int)c.Kp, each, hc, c.Tp * c.Kp);
    else ce_prepare_kernel<true, false><<<grid, 256, 0, st>>>(tk, h, ldh, (int)H, (int)c.Kp, each, hc, c.Tp * c.Kp);
  } else {
    if (scan) ce_prepare_kernel<false, true><<<grid, 256, 0, st>>>(tk, h, ldh, (int)H, (int)c.Kp, each, hc, c.Tp * c.Kp);
    else ce_prepare_kernel<false, false><<<grid, 256, 0, st>>>(tk, h, ldh, (int)H, (int)c.Kp, each, hc, c.Tp * c.Kp);
  }
  CEEG_CHECK_LAUNCH();
  const CeMat Bm{hc, c.Kp, c.Tp * c.Kp, 0, nullptr, INT_MAX};
  for (int p = 0; p < c.pieces; ++p) {
    const int64_t v0 = p * c.piece, Vc = V - v0 < c.piece ? V - v0 : c.piece;
    CeMat A{static_cast<const unsigned short*>(W) + v0 * ldw, ldw, 0, (int)Vc, nullptr, INT_MAX};
    if (!c.direct) {
      ce_pack(dtype, ce_at(W, v0 * ldw, dtype), ldw, Vc, H, c.Kp, false, wc, c.piece * c.Kp, st);
      CEEG_CHECK_LAUNCH();
      A = CeMat{wc, c.Kp, c.piece * c.Kp, (int)Vc, nullptr, INT_MAX};
    }
    const unsigned grid = (unsigned)ce_tiles(c.P, c.e_logits, Vc, T);
#define CE_CALL(PL, BM, BN, WM, WN, TILE) \
  ce_stats_kernel<CE_TILE_OF(TILE), PL, BM, BN, WM, WN><<<grid, WM * WN * 64, 0, st>>>(A, Bm, n, yc, (int)v0, (int)c.Kp, (int)(v0 / BM), parts, part, at_y)
    CE_TILES(c.P, c.e_logits, false, false, CE_CALL);
#undef CE_CALL
    CEEG_CHECK_LAUNCH();
  }
  ce_lse_kernel<<<(unsigned)((T + 3) / 4), 256, 0, st>>>(n, part, parts, at_y, yc, reduction == 0 ? rows : nullptr, lse, reduction == 0 ? loss : rowloss);
  CEEG_CHECK_LAUNCH();
  if (reduction != 0) {
    ce_loss_kernel<<<1, 1024, 0, st>>>(n, rowloss, reduction, loss);
    CEEG_CHECK_LAUNCH();
  }
  return CEEG_OK;
}

extern "C" int ceeg_linear_ce_bwd(const void* packed, const void* W, int64_t ldw, int64_t T, int64_t H, int64_t V, int dtype, int reduction, const float* g, const float* lse,
                                  const int32_t* tokens, void* dh, void* dw, void* ws, size_t ws_bytes, void* stream) {
  const int rc = ce_check(packed, H, W, ldw, T, H, V, dtype);
  if (rc) return rc;
  if (!ceeg_aligned(packed, 256)) return CEEG_EINVAL;
  if (!g || !lse || !tokens || (!dh && !dw) || reduction < 0 || reduction > 2) return CEEG_EINVAL;
  if (!ws || !ceeg_aligned(ws, 256) || ws_bytes < ce_bwd_bytes(T, H, V, dtype)) return CEEG_EWORKSPACE;
  const CePlan c = ce_plan(T, H, V, dtype, true);
  CeegWs w(ws, ws_bytes);
  const unsigned short* const hc = static_cast<const unsigned short*>(packed);
  unsigned short* wc = c.direct ? nullptr : w.take<unsigned short>((size_t)c.P * c.piece * c.Kp);
  unsigned short* tail = c.direct ? w.take<unsigned short>((size_t)PAD * c.Kp) : nullptr;
  unsigned short* dl = w.take<unsigned short>((size_t)c.P * c.Tp * c.ldv);
  float* dh_slots = w.take<float>((size_t)c.dh_cut.room * H);
  float* dw_slots = c.dw_slots > 1 ? w.take<float>((size_t)c.dw_slots * c.piece * H) : nullptr;
  float* top = w.take<float>(1);
  float* r = w.take<float>(T);
  if (!w.ok) return CEEG_EWORKSPACE;
  const int32_t *n = tokens, *rows = tokens + 1, *pos = rows + T, *yc = pos + T;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const CeScale scale{g, reduction, top, r};
  if (reduction == 0) {
    ce_scale_kernel<<<1, 1024, 0, st>>>(n, rows, g, top, r);
    CEEG_CHECK_LAUNCH();
  }
  const CeMat hm{hc, c.Kp, c.Tp * c.Kp, 0, nullptr, INT_MAX}, hk{hc, c.Kp, c.Tp * c.Kp, (int)c.Kp, nullptr, INT_MAX};
  for (int p = 0; p < c.pieces; ++p) {
    const int64_t v0 = p * c.piece, Vc = V - v0 < c.piece ? V - v0 : c.piece, ldv = up(Vc, PAD), plane = c.Tp * c.ldv;
    CeMat A{static_cast<const unsigned short*>(W) + v0 * ldw, ldw, 0, (int)Vc, nullptr, INT_MAX};
    if (!c.direct) {
      ce_pack(dtype, ce_at(W, v0 * ldw, dtype), ldw, Vc, H, c.Kp, true, wc, c.piece * c.Kp, st);
      CEEG_CHECK_LAUNCH();
      A = CeMat{wc, c.Kp, c.piece * c.Kp, (int)Vc, nullptr, INT_MAX};
    }
    const unsigned grid_l = (unsigned)ce_tiles(c.P, c.e_logits, ldv, T);
#define CE_CALL(PL, BM, BN, WM, WN, TILE)                                                                                                                                     \
  ce_dlogits_kernel<CE_TILE_OF(TILE), PL, BM, BN, WM, WN><<<grid_l, WM * WN * 64, 0, st>>>(A, hm, n, yc, lse, scale, (int)v0, (int)ldv, plane, (int)c.Kp, dl)
    CE_TILES(c.P, c.e_logits, false, false, CE_CALL);
#undef CE_CALL
    CEEG_CHECK_LAUNCH();
    if (dh) {
      const CeMat Wk{A.p, A.ld, A.plane, (int)c.Kp, tail, c.direct && Vc % PAD ? (int)(Vc / PAD * PAD) : INT_MAX}, dlm{dl, ldv, plane, 0, nullptr, INT_MAX};
      if (Wk.k_tail != INT_MAX) {
        ce_pack(dtype, ce_at(W, (v0 + Wk.k_tail) * ldw, dtype), ldw, Vc % PAD, H, c.Kp, true, tail, 0, st);
        CEEG_CHECK_LAUNCH();
      }
      const int all = (int)ce_tiles(c.P, c.e_dh, H, T), grid = all > c.dh_cut.want ? all : c.dh_cut.want;  // one stretch of every tile, or as many as are wanted
#define CE_CALL(PL, BM, BN, WM, WN, TILE)                                                                                                                                              \
  ce_slots_kernel<CE_TILE_OF(TILE), BM, BN, WM, WN><<<grid, WM * WN * 64, 0, st>>>(Wk, dlm, n, 1, (int)H, T, (int)ldv, (int)c.ldv, c.dh_cut, p > 0, dh_slots)
      CE_TILES(c.P, c.e_dh, true, false, CE_CALL);
#undef CE_CALL
      CEEG_CHECK_LAUNCH();
    }
    if (dw) {
      const CeMat dlk{dl, ldv, plane, (int)ldv, nullptr, INT_MAX};
      const int all = (int)ce_tiles(c.P, c.e_dw, H, Vc);
      void* const to = const_cast<void*>(ce_at(dw, v0 * H, dtype));
      if (c.dw_slots > 1) {
#define CE_CALL(PL, BM, BN, WM, WN, TILE)                                                                                                                                      \
  ce_slots_kernel<CE_TILE_OF(TILE), BM, BN, WM, WN><<<all * c.dw_slots, WM * WN * 64, 0, st>>>(hk, dlk, n, 0, (int)H, Vc, 0, 0, CeCut{0, c.dw_slots, 0}, 0, dw_slots)
        CE_TILES(c.P, c.e_dw, true, true, CE_CALL);
#undef CE_CALL
        CEEG_CHECK_LAUNCH();
        const unsigned grid = (unsigned)((Vc * H + 255) / 256);
        if (dtype == CEEG_F32) ce_dw_join_kernel<true><<<grid, 256, 0, st>>>(dw_slots, c.dw_slots, n, scale, Vc * H, to);
        else ce_dw_join_kernel<false><<<grid, 256, 0, st>>>(dw_slots, c.dw_slots, n, scale, Vc * H, to);
      } else {
#define CE_CALL(PL, BM, BN, WM, WN, TILE) ce_dw_kernel<CE_TILE_OF(TILE), PL == 3, BM, BN, WM, WN><<<all, WM * WN * 64, 0, st>>>(hk, dlk, n, scale, (int)H, (int)Vc, to)
        CE_TILES(c.P, c.e_dw, true, true, CE_CALL);
#undef CE_CALL
      }
      CEEG_CHECK_LAUNCH();
    }
  }
  if (dh) {
    const unsigned grid = (unsigned)((T * ((H + 3) / 4) + 255) / 256);
    if (dtype == CEEG_F32) ce_dh_join_kernel<true><<<grid, 256, 0, st>>>(dh_slots, c.P, c.e_dh, (int)c.ldv, c.dh_cut, n, pos, scale, T, (int)H, dh);
    else ce_dh_join_kernel<false><<<grid, 256, 0, st>>>(dh_slots, c.P, c.e_dh, (int)c.ldv, c.dh_cut, n, pos, scale, T, (int)H, dh);
    CEEG_CHECK_LAUNCH();
  }
  return CEEG_OK;
}
