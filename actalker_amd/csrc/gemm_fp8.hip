// Matrix product of e4m3 values with a scale for each block of 128:
//
//   C[m][n] = sum_b as[m][b] ws[n / 128][b] sum_{k in block b} A[m][k] W[n][k]  (+ bias[n] + R[m][n])
//
// One v_mfma_f32_16x16x128_f8f6f4 covers exactly one block of k, so the scales never enter the matrix unit: each
// product starts from zero and is added to the fp32 accumulators by one multiply-add a value with the two scales'
// product. The instruction takes W's rows as its first operand, so a lane's four results are four consecutive columns
// n of one row m: as[m] is one value a lane, ws one value a tile, and outputs leave as packed rows.
//
// Precision. The 8-bit matrix instructions add products in groups of 8 consecutive k and drop what lies below 2^-13 of
// the group's largest product (toward zero; measured on the card lane by lane, the same for the 32-deep form), which
// costs up to 7 * 2^-13 of a group's largest product and in practice 2e-6 (signed) to 3e-6 (positive data) of the sum
// of magnitudes. Tiles of many rows with 16-bit outputs, which the matrix rate bounds, take that: 2.7e-5 of the output's
// norm beside the 1.66e-3 (bf16) or 2.1e-4 (fp16) of its own rounding (16384 x 2560 x 5120: distance from the 64-bit
// result 1.65572e-3, of that result rounded 1.65566e-3; fp16 2.0750e-4 and 2.0700e-4). fp32 outputs would show it
// (1.8e-5 of their norm), and few rows, which the weights' bytes bound, gain little by it: those products go through
// the 16-bit matrix instructions, where e4m3 values are exact and the same sums are off by 1e-9 to 1e-8, at half the rate.
#include "gemm_common.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// 16 x 16 x 128: a lane gives row lane % 16 and 32 bytes of k of each operand; the same bytes are taken from both, so
// which 32 a lane takes does not matter
__device__ __forceinline__ f32x4_t mfma8(i32x8_t a, i32x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8_t frag(const char* lds, int at0, int at1) {
  const int4 lo = *reinterpret_cast<const int4*>(lds + at0);
  const int4 hi = *reinterpret_cast<const int4*>(lds + at1);
  return (i32x8_t){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}

// the 16-bit forms of 8 bytes, exactly
__device__ __forceinline__ bf16x8_t wide8(int x0, int x1) {
  bf16x8_t o;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int x = w ? x1 : x0;
#if ACTH_F16
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true);
#else
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true);
#endif
    o[4 * w] = lo[0]; o[4 * w + 1] = lo[1]; o[4 * w + 2] = hi[0]; o[4 * w + 3] = hi[1];
  }
  return o;
}

// bias, residual and store of four consecutive columns [n, n + 4) of row m
__device__ __forceinline__ void finish4(const ActhGemmFp8Desc& p, int m, int n, f32x4_t v, int vec) {
  if (m >= p.M) return;
  if (vec && n + 4 <= p.N) {
    if (p.bias) {
      const float4 b = *reinterpret_cast<const float4*>(p.bias + n);
      v[0] += b.x; v[1] += b.y; v[2] += b.z; v[3] += b.w;
    }
    if (p.R) {
      const uint2 r = *reinterpret_cast<const uint2*>((const bf16_t*)p.R + m * p.ldr + n);
      v[0] += lo16f(r.x); v[1] += hi16f(r.x); v[2] += lo16f(r.y); v[3] += hi16f(r.y);
    }
    if (p.out_f32) *reinterpret_cast<float4*>((float*)p.C + m * p.ldc + n) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>((bf16_t*)p.C + m * p.ldc + n) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= p.N) break;
    float x = v[i];
    if (p.bias) x += p.bias[n + i];
    if (p.R) x += bf2f(((const bf16_t*)p.R)[m * p.ldr + n + i]);
    if (p.out_f32) ((float*)p.C)[m * p.ldc + n + i] = x;
    else ((bf16_t*)p.C)[m * p.ldc + n + i] = f2bf(x);
  }
}

__device__ __forceinline__ int4 load16_whole(const uint8_t* p) {
  struct __attribute__((packed, aligned(1))) Any { int v[4]; };
  const Any a = *reinterpret_cast<const Any*>(p);
  return make_int4(a.v[0], a.v[1], a.v[2], a.v[3]);
}

// bytes [k, k + 16) of a row of K bytes at any address, zeros behind its end: one unaligned load. A piece that the end
// cuts is loaded from 16 bytes before the end and moved down, so nothing behind the row is read.
__device__ __forceinline__ int4 load16_any(const uint8_t* row, int k, int K) {
  struct __attribute__((packed, aligned(1))) Any { unsigned long long v[2]; };
  if (k >= K) return make_int4(0, 0, 0, 0);
  unsigned long long lo = 0, hi = 0;
  if (k + 16 <= K) {
    const Any a = *reinterpret_cast<const Any*>(row + k);
    lo = a.v[0]; hi = a.v[1];
  } else if (K >= 16) {
    const Any a = *reinterpret_cast<const Any*>(row + K - 16);
    const int s = (16 - (K - k)) * 8;              // 8 .. 120 bits
    lo = s < 64 ? (a.v[0] >> s) | (a.v[1] << (64 - s)) : a.v[1] >> (s - 64);
    hi = s < 64 ? a.v[1] >> s : 0;
  } else {
#pragma unroll
    for (int e = 0; e < 15; ++e)
      if (k + e < K) {
        if (e < 8) lo |= (unsigned long long)row[k + e] << (8 * (e & 7));
        else hi |= (unsigned long long)row[k + e] << (8 * (e & 7));
      }
  }
  return make_int4((int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32));
}

// ---- large tiles: BM x BN, eight waves of TM x TN fragments, one k block (128 bytes a row) a step, double-buffered
// LDS-DMA. 16-byte chunk c of row r lies at chunk c ^ (r % 8) of its 128-byte LDS row, so the 8 lanes of a ds_read_b128
// group, which read one chunk of 8 rows, meet 8 different bank slots; the DMA, whose LDS side is linear, applies the
// same exchange to its global side.
// Bound: 8192^3 takes 531 us (2070 TFLOP/s; the card's library reaches 2690 to 3230, by data and card, with one scale for a
// whole operand, 1250 to 1590 in 16 bits). Counters at 16384 x 2560 x 5120: the matrix unit is busy 40 % of the time, the vector
// unit, with the scales' multiply-adds, 36 %, the LDS reads 19 % without a conflict; the waves stand at the end of a block 41 %
// of their time and wait for an issue slot 29 %. So it is the one barrier a block, behind the LDS-DMA, that two waves a SIMD
// cannot cover (17 % of the time goes to the DMA beside the products and 5 % to the multiply-adds, both timed by leaving them out
// of a copy). Then rounds of 256 tiles: 16384 x 2560 is 2.5 of them, the last taken as a round of half tiles, at 0.65 of a
// round's time (215 - 240 us, 1790 - 2000 TFLOP/s at K = 5120; a ring of three 256 x 128 stages, five full rounds there, moves
// twice the bytes a product through L2 and took 275).
template <int BM, int BN>
struct Tile {
  static constexpr int WC = BN / 64, WR = 8 / WC;              // waves along n and m
  static constexpr int TM = BM / WR / 16, TN = 4;              // fragments of a wave
  static constexpr int AB = BM * 128, STAGE = (BM + BN) * 128;
  static constexpr int AP = BM / 64, WP = BN / 64;             // DMA pieces of 8 rows a wave and step
};

}  // namespace

// One step: the DMA of the next k block into `wr`, the products of the block in `rd`. The two stage buffers come in as
// restricted pointers of their own: told apart, the reads of one need not wait for the loads into the other (the
// compiler otherwise drains all LDS-DMA before every ds_read).
template <int BM, int BN>
struct Stage {
  using T = Tile<BM, BN>;
  __amdgpu_buffer_rsrc_t ra, rw, rs;
  unsigned oa[T::AP], ow[T::WP], os;
  int wave, chunk, K;
  long long as_blk;

  __device__ __forceinline__ void dma(char* wr, int kb) const {
    const bool dead = kb * 128 + chunk * 16 >= K;
#pragma unroll
    for (int u = 0; u < T::AP; ++u)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void*)(wr + (wave + 8 * u) * 1024), 16, dead ? gemm::OOB : oa[u], kb * 128, 0, 0);
#pragma unroll
    for (int u = 0; u < T::WP; ++u)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_void*)(wr + T::AB + (wave + 8 * u) * 1024), 16, dead ? gemm::OOB : ow[u], kb * 128, 0, 0);
    if (wave < BM / 64)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(wr + T::AB + BN * 128 + wave * 256), 4, os, (int)(kb * as_blk * 4), 0, 0);
  }
};

// workgroup b of nwg takes this place of the tiles' order: each XCD a contiguous run
__device__ __forceinline__ int place_of(int b, int nwg) {
  const int xcd = b & 7, qn = nwg >> 3, rn = nwg & 7;
  return (xcd < rn ? xcd * (qn + 1) : rn * (qn + 1) + (xcd - rn) * qn) + (b >> 3);
}

// the tiles' order: gm row blocks x all column blocks, rows fastest, so the tiles that an XCD holds at once share their
// rows of A and W in its L2
template <int BM, int BN>
__device__ __forceinline__ void tile_at(const ActhGemmFp8Desc& p, int gm, int lin, int& m0, int& n0) {
  const int ntn = (p.N + BN - 1) / BN, ntm = (p.M + BM - 1) / BM;
  const int grp = lin / (gm * ntn), mg0 = grp * gm, gcur = min(gm, ntm - mg0), rest = lin - grp * gm * ntn;
  n0 = rest / gcur * BN;
  m0 = (mg0 + rest % gcur) * BM;
}

// Products run LAG ahead of the multiply-adds that take them in, in exactly this order (sched_barrier): the matrix unit
// then never waits for the vector unit's use of its last result. LAG 1, 2, 3, 4, 8: 571, 546, 531, 528, 528 us at 8192^3.
constexpr int LAG = 3;

template <int BM, int BN, bool WIDE>
__device__ __forceinline__ void step(const char* __restrict__ rd, char* __restrict__ wr, const Stage<BM, BN>& st, int next, bool more,
                                     int a_row, int w_row, int s_row, int f0, int f1, float ws,
                                     f32x4_t (&acc)[Tile<BM, BN>::TM][Tile<BM, BN>::TN]) {
  using T = Tile<BM, BN>;
  i32x8_t fw[T::TN], fa[2];
  float sc[T::TM];
  fa[0] = frag(rd, a_row + f0, a_row + f1);
#pragma unroll
  for (int j = 0; j < T::TN; ++j) fw[j] = frag(rd, w_row + j * 2048 + f0, w_row + j * 2048 + f1);
#pragma unroll
  for (int i = 0; i < T::TM; ++i) sc[i] = *reinterpret_cast<const float*>(rd + s_row + i * 64) * ws;
  if (more) st.dma(wr, next);
  f32x4_t d[LAG + 1];
#pragma unroll
  for (int t = 0; t < T::TM * T::TN + LAG; ++t) {
    const int i = t / T::TN, j = t % T::TN;
    if (t < T::TM * T::TN) {
      if (j == 0 && i + 1 < T::TM) fa[(i + 1) & 1] = frag(rd, a_row + (i + 1) * 2048 + f0, a_row + (i + 1) * 2048 + f1);
      if constexpr (WIDE) {
        f32x4_t v = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c)
          v = mfma16x16x32(wide8(fw[j][2 * c], fw[j][2 * c + 1]), wide8(fa[i & 1][2 * c], fa[i & 1][2 * c + 1]), v);
        d[t % (LAG + 1)] = v;
      } else {
        d[t % (LAG + 1)] = mfma8(fw[j], fa[i & 1], (f32x4_t){0, 0, 0, 0});
      }
    }
    if (t >= LAG) {
      const int u = t - LAG;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[u / T::TN][u % T::TN][e] = fmaf(d[u % (LAG + 1)][e], sc[u / T::TN], acc[u / T::TN][u % T::TN][e]);
    }
    if (!WIDE) __builtin_amdgcn_sched_barrier(0);
  }
}

constexpr int MAXKB = 1024;
template <int BM, int BN>                          // two stages (rows of A, of W, and the row scales), W's scales
constexpr int lds_bytes() { return 2 * (Tile<BM, BN>::STAGE + BM * 4) + MAXKB * (BN / 128) * 4; }

template <int BM, int BN, bool WIDE>
__device__ __forceinline__ void gemm_fp8_tile(const ActhGemmFp8Desc& p, int m0, int n0, int vec_out, char* smem) {
  using T = Tile<BM, BN>;
  constexpr int STAGE = T::STAGE + BM * 4;
  float* const s_ws = reinterpret_cast<float*>(smem + 2 * STAGE);             // [kb][BN / 128]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % T::WR, wc = wave / T::WR;
  const int r16 = lane & 15, g = lane >> 4;
  const int nkb = (p.K + 127) / 128;

  const int mrows = min(BM, p.M - m0), nrows = min(BN, p.N - n0);
  Stage<BM, BN> st;
  st.ra = gemm::make_rsrc((const uint8_t*)p.A + (long long)m0 * p.lda, (unsigned)((mrows - 1) * p.lda + p.K));
  st.rw = gemm::make_rsrc((const uint8_t*)p.W + (long long)n0 * p.ldw, (unsigned)((nrows - 1) * p.ldw + p.K));
  st.rs = gemm::make_rsrc(p.ascale + (long long)m0 * p.as_row, 0x7fffffffu);
  st.wave = wave; st.chunk = (lane & 7) ^ (lane >> 3); st.K = p.K; st.as_blk = p.as_blk;
#pragma unroll
  for (int u = 0; u < T::AP; ++u) {
    const int r = (wave + 8 * u) * 8 + (lane >> 3);
    st.oa[u] = r < mrows ? (unsigned)(r * p.lda + st.chunk * 16) : gemm::OOB;
  }
#pragma unroll
  for (int u = 0; u < T::WP; ++u) {
    const int r = (wave + 8 * u) * 8 + (lane >> 3);
    st.ow[u] = r < nrows ? (unsigned)(r * p.ldw + st.chunk * 16) : gemm::OOB;
  }
  st.os = (unsigned)(min(wave * 64 + lane, mrows - 1) * p.as_row * 4);

  f32x4_t acc[T::TM][T::TN];
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};

  st.dma(smem, 0);
  for (int i = tid; i < nkb * (BN / 128); i += 512) {
    const int kb = i / (BN / 128), nb = n0 / 128 + i % (BN / 128);
    s_ws[i] = nb * 128 < p.N ? p.wscale[(long long)nb * p.ws_row + kb * p.ws_blk] : 0.0f;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  const int f0 = (g ^ (r16 & 7)) * 16, f1 = ((g + 4) ^ (r16 & 7)) * 16;
  const int a_row = (wr * T::TM * 16 + r16) * 128, w_row = T::AB + (wc * 64 + r16) * 128;
  const int s_row = T::STAGE + (wr * T::TM * 16 + r16) * 4;
  for (int kb = 0; kb < nkb; ++kb) {
    const float ws = s_ws[kb * (BN / 128) + wc * 64 / 128];
    step<BM, BN, WIDE>(smem + (kb & 1) * STAGE, smem + (~kb & 1) * STAGE, st, kb + 1, kb + 1 < nkb, a_row, w_row, s_row, f0, f1, ws, acc);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
      finish4(p, m0 + (wr * T::TM + i) * 16 + r16, n0 + wc * 64 + j * 16 + g * 4, acc[i][j], vec_out);
}

template <bool WIDE>
__global__ __launch_bounds__(512, WIDE ? 2 : 4) void gemm_fp8_kernel(const ActhGemmFp8Desc p, int gm, int vec_out) {
  __shared__ __attribute__((aligned(16))) char smem[lds_bytes<128, 128>()];
  int m0, n0;
  tile_at<128, 128>(p, gm, place_of(blockIdx.x, gridDim.x), m0, n0);
  gemm_fp8_tile<128, 128, WIDE>(p, m0, n0, vec_out, smem);
}

// 256 x 256 tiles, the first `whole` of them by a workgroup each, the others in halves of 128 columns
__global__ __launch_bounds__(512, 2) void gemm_fp8_large_kernel(const ActhGemmFp8Desc p, int gm, int whole, int vec_out) {
  __shared__ __attribute__((aligned(16))) char smem[lds_bytes<256, 256>()];
  int m0, n0;
  if ((int)blockIdx.x < whole) {
    tile_at<256, 256>(p, gm, place_of(blockIdx.x, whole), m0, n0);
    gemm_fp8_tile<256, 256, false>(p, m0, n0, vec_out, smem);
  } else {
    const int at = place_of(blockIdx.x - whole, gridDim.x - whole);
    tile_at<256, 256>(p, gm, whole + (at >> 1), m0, n0);
    n0 += (at & 1) * 128;
    if (n0 < p.N) gemm_fp8_tile<256, 128, false>(p, m0, n0, vec_out, smem);
  }
}

// The 128 x 128 tile for operands that the LDS-DMA cannot take (rows at any address, a K that ends inside 16 bytes, very
// long rows): the next block goes through registers, loaded before this one's products and written to LDS after them.
// One block a CU: held to the 128 registers of two it spills (4096 x 2560 x 2561: 118 against 98 us; fp32 outputs of the
// DMA tile likewise, 4096 x 2560 x 2560: 127 against 78 us).
template <bool WIDE>
__global__ __launch_bounds__(512, 2) void gemm_fp8_any_kernel(const ActhGemmFp8Desc p, int gm, int vec_out) {
  constexpr int BM = 128, BN = 128;
  using T = Tile<BM, BN>;
  constexpr int STAGE = T::STAGE + BM * 4;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % T::WR, wc = wave / T::WR;
  const int r16 = lane & 15, g = lane >> 4;
  int m0, n0;
  tile_at<BM, BN>(p, gm, place_of(blockIdx.x, gridDim.x), m0, n0);
  const int nkb = (p.K + 127) / 128;
  const int chunk = (lane & 7) ^ (lane >> 3);
  const uint8_t* ar[T::AP];
  const uint8_t* wrow[T::WP];
#pragma unroll
  for (int u = 0; u < T::AP; ++u) ar[u] = (const uint8_t*)p.A + min(m0 + (wave + 8 * u) * 8 + (lane >> 3), p.M - 1) * p.lda;
#pragma unroll
  for (int u = 0; u < T::WP; ++u) wrow[u] = (const uint8_t*)p.W + min(n0 + (wave + 8 * u) * 8 + (lane >> 3), p.N - 1) * p.ldw;
  const float* const as = p.ascale + min(m0 + tid % BM, p.M - 1) * p.as_row;
  const float* const ws = p.wscale + (long long)(n0 >> 7) * p.ws_row;
  int4 ra[T::AP], rw[T::WP];
  float rs = 0.0f;
  auto load = [&](int kb) {
    const int k = kb * 128 + chunk * 16;
    if (kb * 128 + 128 <= p.K) {                   // a whole block
#pragma unroll
      for (int u = 0; u < T::AP; ++u) ra[u] = load16_whole(ar[u] + k);
#pragma unroll
      for (int u = 0; u < T::WP; ++u) rw[u] = load16_whole(wrow[u] + k);
    } else {
#pragma unroll
      for (int u = 0; u < T::AP; ++u) ra[u] = load16_any(ar[u], k, p.K);
#pragma unroll
      for (int u = 0; u < T::WP; ++u) rw[u] = load16_any(wrow[u], k, p.K);
    }
    rs = as[kb * p.as_blk];
  };
  auto store = [&](char* to) {
#pragma unroll
    for (int u = 0; u < T::AP; ++u) *reinterpret_cast<int4*>(to + (wave + 8 * u) * 1024 + lane * 16) = ra[u];
#pragma unroll
    for (int u = 0; u < T::WP; ++u) *reinterpret_cast<int4*>(to + T::AB + (wave + 8 * u) * 1024 + lane * 16) = rw[u];
    if (tid < BM) *reinterpret_cast<float*>(to + T::STAGE + tid * 4) = rs;
  };

  f32x4_t acc[T::TM][T::TN];
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};

  load(0);
  store(smem);
  __syncthreads();
  const int f0 = (g ^ (r16 & 7)) * 16, f1 = ((g + 4) ^ (r16 & 7)) * 16;
  const int a_row = (wr * T::TM * 16 + r16) * 128, w_row = T::AB + (wc * 64 + r16) * 128;
  const int s_row = T::STAGE + (wr * T::TM * 16 + r16) * 4;
  const Stage<BM, BN> none = {};
  for (int kb = 0; kb < nkb; ++kb) {
    const bool more = kb + 1 < nkb;
    if (more) load(kb + 1);
    step<BM, BN, WIDE>(smem + (kb & 1) * STAGE, nullptr, none, 0, false, a_row, w_row, s_row, f0, f1, ws[kb * p.ws_blk], acc);
    if (more) store(smem + (~kb & 1) * STAGE);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
      finish4(p, m0 + (wr * T::TM + i) * 16 + r16, n0 + wc * 64 + j * 16 + g * 4, acc[i][j], vec_out);
}

template __global__ void gemm_fp8_kernel<false>(const ActhGemmFp8Desc, int, int);
template __global__ void gemm_fp8_kernel<true>(const ActhGemmFp8Desc, int, int);
template __global__ void gemm_fp8_any_kernel<false>(const ActhGemmFp8Desc, int, int);
template __global__ void gemm_fp8_any_kernel<true>(const ActhGemmFp8Desc, int, int);

namespace {

// ---- few rows: a tile of 16 MT x 16 NT, its k blocks dealt to the eight waves in turn (few rows make few tiles, so the
// long axis has to fill the chip), each wave's fragments straight from memory: no wave waits for another until the
// partial sums meet in LDS, in a fixed order. A lane loads two 16-byte pieces of its row, k [16 g, 16 g + 16) and 64
// further. Rows behind the last read it again. The sums go through the 16-bit unit, exact to fp32's roundings; the 8-bit one
// would save 4 to 20 % where a wave takes three blocks or more (32 columns a workgroup: 1 x 2560 x 2560 5.5 against 6.5 us,
// 1 x 5120 x 640 3.6 and 3.7).
// Bound: the weights' bytes and the latency of the two or three blocks each wave takes (1 x 10240 x 2560 from memory: 10.7
// us, 2.5 TB/s; 1 x 2560 x 2560: 6.6 us; two or four blocks' loads at once changed neither), then L2, which serves A and W
// to every tile: larger row counts take larger tiles.
template <int MT, int NT, bool ALIGNED>
__global__ __launch_bounds__(512, MT * NT >= 8 ? 2 : 4) void gemm_fp8_few_kernel(const ActhGemmFp8Desc p, int vec_out) {
  constexpr int TILES = MT * NT;
  __shared__ __attribute__((aligned(16))) f32x4_t red[4][TILES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int ntm = (p.M + 16 * MT - 1) / (16 * MT);
  const int m0 = (int)(blockIdx.x % ntm) * 16 * MT, n0 = (int)(blockIdx.x / ntm) * 16 * NT;
  const int nkb = (p.K + 127) / 128;
  const int mrows = min(16 * MT, p.M - m0), nrows = min(16 * NT, p.N - n0);
  const __amdgpu_buffer_rsrc_t ra = gemm::make_rsrc((const uint8_t*)p.A + (long long)m0 * p.lda, (unsigned)((mrows - 1) * p.lda + p.K));
  const __amdgpu_buffer_rsrc_t rw = gemm::make_rsrc((const uint8_t*)p.W + (long long)n0 * p.ldw, (unsigned)((nrows - 1) * p.ldw + p.K));
  unsigned oa[MT], ow[NT];                         // ALIGNED: offsets in the buffers above; else row pointers
  const uint8_t *pa[MT], *pw[NT];
  const float* as[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = min(i * 16 + r16, mrows - 1);
    oa[i] = (unsigned)(r * p.lda + g * 16);
    pa[i] = (const uint8_t*)p.A + (long long)(m0 + r) * p.lda;
    as[i] = p.ascale + (long long)(m0 + r) * p.as_row;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = min(j * 16 + r16, nrows - 1);
    ow[j] = (unsigned)(r * p.ldw + g * 16);
    pw[j] = (const uint8_t*)p.W + (long long)(n0 + r) * p.ldw;
  }
  const float* const wsp = p.wscale + (long long)(n0 >> 7) * p.ws_row;       // 16 NT divides 128: one block of columns

  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};

  typedef int i32x4_t __attribute__((ext_vector_type(4)));
  i32x4_t fa[MT][2], fw[NT][2];
  for (int kb = wave; kb < nkb; kb += 8) {
    const int k0 = kb * 128;
    const bool in0 = k0 + g * 16 < p.K, in1 = k0 + 64 + g * 16 < p.K;      // pieces behind K: zeros
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if constexpr (ALIGNED) {
        fw[j][0] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, in0 ? ow[j] : gemm::OOB, k0, 0));
        fw[j][1] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, in1 ? ow[j] + 64 : gemm::OOB, k0, 0));
      } else {
        fw[j][0] = __builtin_bit_cast(i32x4_t, load16_any(pw[j], k0 + g * 16, p.K));
        fw[j][1] = __builtin_bit_cast(i32x4_t, load16_any(pw[j], k0 + 64 + g * 16, p.K));
      }
    }
    float sc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (ALIGNED) {
        fa[i][0] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ra, in0 ? oa[i] : gemm::OOB, k0, 0));
        fa[i][1] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ra, in1 ? oa[i] + 64 : gemm::OOB, k0, 0));
      } else {
        fa[i][0] = __builtin_bit_cast(i32x4_t, load16_any(pa[i], k0 + g * 16, p.K));
        fa[i][1] = __builtin_bit_cast(i32x4_t, load16_any(pa[i], k0 + 64 + g * 16, p.K));
      }
      sc[i] = as[i][kb * p.as_blk];
    }
    const float ws = wsp[kb * p.ws_blk];
    f32x4_t d[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) d[i][j] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      bf16x8_t wa[MT], ww[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) wa[i] = wide8(fa[i][c >> 1][(c & 1) * 2], fa[i][c >> 1][(c & 1) * 2 + 1]);
#pragma unroll
      for (int j = 0; j < NT; ++j) ww[j] = wide8(fw[j][c >> 1][(c & 1) * 2], fw[j][c >> 1][(c & 1) * 2 + 1]);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) d[i][j] = mfma16x16x32(ww[j], wa[i], d[i][j]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float s = sc[i] * ws;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[i][j][e], s, acc[i][j][e]);
    }
  }

  // waves 4 .. 7 to 0 .. 3, then every wave sums its share of the tiles over the four
  if (wave >= 4) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) red[wave - 4][t][lane] = acc[t / NT][t % NT];
  }
  __syncthreads();
  if (wave < 4) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) red[wave][t][lane] += acc[t / NT][t % NT];
  }
  __syncthreads();
  for (int t = wave; t < TILES; t += 8) {
    const f32x4_t v = (red[0][t][lane] + red[1][t][lane]) + (red[2][t][lane] + red[3][t][lane]);
    finish4(p, m0 + t / NT * 16 + r16, n0 + t % NT * 16 + g * 4, v, vec_out);
  }
}

template <bool ALIGNED>
void launch_few(const ActhGemmFp8Desc& d, int vec_out, hipStream_t stream) {
  auto tiles = [&](int mt, int nt) { return (unsigned)(((d.M + 16 * mt - 1) / (16 * mt)) * ((d.N + 16 * nt - 1) / (16 * nt))); };
  // 32 columns a workgroup against 64, up to 16 rows (weights from memory, a call in a graph): 1 x 2560 x 2560 6.6 against
  // 9.8 us, 1 x 10240 x 2560 10.7 against 11.6, 1 x 16384 x 5120 19.9 against 23.2; 16 rows 7.4 against 11.0, 13.4 against
  // 12.7, 24.8 against 24.2. 32 rows a tile while they leave CUs free: 128 x 2560 x 2560 12.1 against 15.5 us of 64 rows,
  // 128 x 5120 x 2560 23.8 against 17.4.
  if (d.M <= 16) {
    gemm_fp8_few_kernel<1, 2, ALIGNED><<<tiles(1, 2), 512, 0, stream>>>(d, vec_out);
  } else if (d.M <= 32 || tiles(4, 4) < 128) {
    gemm_fp8_few_kernel<2, 4, ALIGNED><<<tiles(2, 4), 512, 0, stream>>>(d, vec_out);
  } else {
    gemm_fp8_few_kernel<4, 4, ALIGNED><<<tiles(4, 4), 512, 0, stream>>>(d, vec_out);
  }
}

bool al(const void* p, long long ld_bytes, int to) { return !p || (((uintptr_t)p | (uintptr_t)ld_bytes) % to) == 0; }

}  // namespace

extern "C" int acth_gemm_fp8(const ActhGemmFp8Desc* d, hipStream_t stream) {
  if (!d || d->M < 0) return ACTH_EINVAL;
  if (d->M == 0) return ACTH_OK;
  if (!d->A || !d->W || !d->C || !d->ascale || !d->wscale || d->N < 1 || d->K < 1) return ACTH_EINVAL;
  if ((d->M > 1 && (d->lda < d->K || d->ldc < d->N || (d->R && d->ldr < d->N))) || (d->N > 1 && d->ldw < d->K))
    return ACTH_EINVAL;
  const int vec_out = al(d->C, d->ldc * (d->out_f32 ? 4 : 2), 16) && al(d->bias, 0, 16) && al(d->R, d->ldr * 2, 8);
  const bool dma = d->K % 16 == 0 && al(d->A, d->lda, 16) && al(d->W, d->ldw, 16) && d->lda < (1 << 22) && d->ldw < (1 << 22) &&
                   d->K <= 128 * 1024 && 256 * d->as_row < (1 << 28) && (d->K + 127) / 128 * d->as_blk < (1 << 28);
  const long long t256 = (long long)((d->M + 255) / 256) * ((d->N + 255) / 256);
  const long long t128 = (long long)((d->M + 127) / 128) * ((d->N + 127) / 128);
  if (d->K > (1 << 30) || d->M > (1 << 30) || d->N > (1 << 27) || t128 >= (1 << 23)) return ACTH_EINVAL;      // a launch: less than 2^32 lanes
  // Rounds of the chip: 256 large tiles in 1.5 times the time of 512 small ones (two blocks a CU). A last round of at most
  // 128 large tiles is taken in halves, in a small round's time. Large against small, in a graph: 4096 x 2560 of K = 640,
  // 2560, 5120, 10240: 21.3 against 19.8 us, 43.4 and 47.2, 72 and 82, 128 and 149; 4096 x 5120: 31.4 and 30.2, 71 and 73, 121 and
  // 129, 224 and 240; 9216 x 2560: 32.4 and 34.4, 73 and 81, 130 and 147, 236 and 274. Halves against whole tiles: 16384 x
  // 2560: 52 and 59, 121 and 132, 215 and 235, 396 and 415. So the rule loses 8 % at most, where K is short.
  const int rest = (int)(t256 % 256), halves = rest <= 128 ? rest : 0;
  const long long large = t256 / 256 * 3 + (halves ? 2 : rest ? 3 : 0), small = (t128 + 511) / 512 * 2;
  // (weights from memory) 256 x 2560 x 2560 15.7 against 22.3 us, 512 rows 28.4 against 24.3; 1024 x 640 x 2560 14.7 against 19.7
  if (d->M <= 32 || t128 <= 40) {
    if (dma) launch_few<true>(*d, vec_out, stream);
    else launch_few<false>(*d, vec_out, stream);
  } else if (!dma) {
    if (d->out_f32) gemm_fp8_any_kernel<true><<<(unsigned)t128, 512, 0, stream>>>(*d, 16, vec_out);
    else gemm_fp8_any_kernel<false><<<(unsigned)t128, 512, 0, stream>>>(*d, 16, vec_out);
  } else if (d->out_f32) {
    gemm_fp8_kernel<true><<<(unsigned)t128, 512, 0, stream>>>(*d, 16, vec_out);
  } else if (large < small) {
    // row blocks side by side: 4, 8, 16, 32: 450, 480, 480, 513 us at 16384 x 10240 x 2560, 249, 256, 256, 257 at 16384 x 2560 x 5120
    gemm_fp8_large_kernel<<<(unsigned)(t256 + halves), 512, 0, stream>>>(*d, 4, (int)(t256 - halves), vec_out);
  } else {
    gemm_fp8_kernel<false><<<(unsigned)t128, 512, 0, stream>>>(*d, 16, vec_out);
  }
  ACTH_CHECK_LAUNCH();
  return ACTH_OK;
}
