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
// of magnitudes: far below a 16-bit output's half step of 2^-9 or 2^-12. fp32 outputs would show it (1.8e-5 of their
// norm), so those products go through the 16-bit matrix instructions instead, where e4m3 values are exact and the same
// sums are off by 1e-9 to 1e-8; that unit runs at half the rate.
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

__device__ __forceinline__ bf16x8_t wide8(const char* lds) {
  const int2 v = *reinterpret_cast<const int2*>(lds);
  return wide8(v.x, v.y);
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

// 16 bytes from any address: one unaligned load
__device__ __forceinline__ int4 load16_any(const uint8_t* p) {
  struct __attribute__((packed, aligned(1))) Any { int v[4]; };
  const Any a = *reinterpret_cast<const Any*>(p);
  return make_int4(a.v[0], a.v[1], a.v[2], a.v[3]);
}

// ---- any sizes, strides and alignment: a 64 x 64 tile, four waves of 32 x 32, one k block at a time through LDS
template <bool WIDE>
__global__ __launch_bounds__(256) void gemm_fp8_any_kernel(const ActhGemmFp8Desc p, int vec_out) {
  constexpr int PITCH = 144;
  __shared__ __align__(16) char sa[64 * PITCH], sw[64 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  const int r16 = lane & 15, g = lane >> 4;
  f32x4_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};

  const int nkb = (p.K + 127) / 128;
  for (int kb = 0; kb < nkb; ++kb) {
    const int k0 = kb * 128;
    // 64 rows x 8 pieces of 16 bytes for each operand
    for (int i = tid; i < 512; i += 256) {
      const int r = i >> 3, c = (i & 7) * 16;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int row = (o ? n0 : m0) + r, rows = o ? p.N : p.M;
        const uint8_t* src = o ? (const uint8_t*)p.W + row * p.ldw : (const uint8_t*)p.A + row * p.lda;
        int4 v = make_int4(0, 0, 0, 0);
        if (row < rows && k0 + c < p.K) {
          if (k0 + c + 16 <= p.K) {
            v = load16_any(src + k0 + c);
          } else {
            uint32_t b[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (k0 + c + e < p.K) b[e >> 2] |= (uint32_t)src[k0 + c + e] << (8 * (e & 3));
            v = make_int4((int)b[0], (int)b[1], (int)b[2], (int)b[3]);
          }
        }
        *reinterpret_cast<int4*>((o ? sw : sa) + r * PITCH + c) = v;
      }
    }
    __syncthreads();
    const float ws = p.wscale[(long long)(n0 >> 7) * p.ws_row + kb * p.ws_blk];
    float sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ra = m0 + wm + i * 16 + r16;
      sc[i] = ra < p.M ? p.ascale[(long long)ra * p.as_row + kb * p.as_blk] * ws : 0.0f;
    }
    f32x4_t d[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) d[i][j] = (f32x4_t){0, 0, 0, 0};
    if constexpr (WIDE) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        bf16x8_t fa[2], fw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fa[i] = wide8(sa + (wm + i * 16 + r16) * PITCH + c * 32 + g * 8);
          fw[i] = wide8(sw + (wn + i * 16 + r16) * PITCH + c * 32 + g * 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) d[i][j] = mfma16x16x32(fw[j], fa[i], d[i][j]);
      }
    } else {
      i32x8_t fa[2], fw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ra = (wm + i * 16 + r16) * PITCH, rw = (wn + i * 16 + r16) * PITCH;
        fa[i] = frag(sa, ra + g * 32, ra + g * 32 + 16);
        fw[i] = frag(sw, rw + g * 32, rw + g * 32 + 16);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) d[i][j] = mfma8(fw[j], fa[i], d[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[i][j][e], sc[i], acc[i][j][e]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) finish4(p, m0 + wm + i * 16 + r16, n0 + wn + j * 16 + g * 4, acc[i][j], vec_out);
}

// ---- large tiles: BM x BN, eight waves of TM x TN fragments, one k block (128 bytes a row) a step, double-buffered
// LDS-DMA. 16-byte chunk c of row r lies at chunk c ^ (r % 8) of its 128-byte LDS row, so the 8 lanes of a ds_read_b128
// group, which read one chunk of 8 rows, meet 8 different bank slots; the DMA, whose LDS side is linear, applies the
// same exchange to its global side.
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

template <int BM, int BN, bool WIDE>
__global__ __launch_bounds__(512, BM * BN > 128 * 128 ? 2 : 4) void gemm_fp8_kernel(const ActhGemmFp8Desc p, int gm, int vec_out) {
  using T = Tile<BM, BN>;
  constexpr int STAGE = T::STAGE + BM * 4;                      // a block's rows of A, of W, and the row scales
  constexpr int MAXKB = 1024;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE + MAXKB * (BN / 128) * 4];
  float* const s_ws = reinterpret_cast<float*>(smem + 2 * STAGE);             // [kb][BN / 128]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % T::WR, wc = wave / T::WR;
  const int r16 = lane & 15, g = lane >> 4;

  // tiles: each XCD takes a contiguous run; inside it gm row blocks x all column blocks, rows fastest
  const int ntn = (p.N + BN - 1) / BN, ntm = (p.M + BM - 1) / BM, nwg = gridDim.x;
  const int xcd = blockIdx.x & 7, qn = nwg >> 3, rn = nwg & 7;
  const int lin = (xcd < rn ? xcd * (qn + 1) : rn * (qn + 1) + (xcd - rn) * qn) + (blockIdx.x >> 3);
  const int grp = lin / (gm * ntn), mg0 = grp * gm, gcur = min(gm, ntm - mg0), rest = lin - grp * gm * ntn;
  const int n0 = rest / gcur * BN, m0 = (mg0 + rest % gcur) * BM;
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


template __global__ void gemm_fp8_kernel<256, 256, false>(const ActhGemmFp8Desc, int, int);
template __global__ void gemm_fp8_kernel<128, 128, false>(const ActhGemmFp8Desc, int, int);
template __global__ void gemm_fp8_kernel<128, 128, true>(const ActhGemmFp8Desc, int, int);

namespace {

// ---- few rows: a tile of 16 MT x 16 NT, its k blocks dealt to the eight waves in turn (few rows make few tiles, so the
// long axis has to fill the chip), each wave's fragments straight from memory: no wave waits for another until the
// partial sums meet in LDS, in a fixed order. A lane loads two 16-byte pieces of its row, k [16 g, 16 g + 16) and 64
// further. Rows behind the last read it again.
// Bound: the weights' bytes and the latency of the two or three blocks each wave takes (1 x 10240 x 2560: 8.5 us, 3.1 TB/s;
// 1 x 2560 x 2560: 5.6 us; two or four blocks' loads at once changed neither), then L2, which serves A and W to every
// tile: larger row counts take larger tiles.
template <int MT, int NT, bool WIDE>
__global__ __launch_bounds__(512, MT * NT > 8 ? 2 : 4) void gemm_fp8_few_kernel(const ActhGemmFp8Desc p, int vec_out) {
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
  unsigned oa[MT], ow[NT];
  const float* as[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = min(i * 16 + r16, mrows - 1);
    oa[i] = (unsigned)(r * p.lda + g * 16);
    as[i] = p.ascale + (long long)(m0 + r) * p.as_row;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) ow[j] = (unsigned)(min(j * 16 + r16, nrows - 1) * p.ldw + g * 16);
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
      fw[j][0] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, in0 ? ow[j] : gemm::OOB, k0, 0));
      fw[j][1] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rw, in1 ? ow[j] + 64 : gemm::OOB, k0, 0));
    }
    float sc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      fa[i][0] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ra, in0 ? oa[i] : gemm::OOB, k0, 0));
      fa[i][1] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ra, in1 ? oa[i] + 64 : gemm::OOB, k0, 0));
      sc[i] = as[i][kb * p.as_blk];
    }
    const float ws = wsp[kb * p.ws_blk];
    f32x4_t d[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) d[i][j] = (f32x4_t){0, 0, 0, 0};
    if constexpr (WIDE) {
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
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          d[i][j] = mfma8(__builtin_shufflevector(fw[j][0], fw[j][1], 0, 1, 2, 3, 4, 5, 6, 7),
                          __builtin_shufflevector(fa[i][0], fa[i][1], 0, 1, 2, 3, 4, 5, 6, 7), d[i][j]);
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

template <bool WIDE>
void launch_few(const ActhGemmFp8Desc& d, int vec_out, hipStream_t stream) {
  auto tiles = [&](int mt, int nt) { return (unsigned)(((d.M + 16 * mt - 1) / (16 * mt)) * ((d.N + 16 * nt - 1) / (16 * nt))); };
  if (d.M <= 16) {
    if (tiles(1, 4) >= 128) gemm_fp8_few_kernel<1, 4, WIDE><<<tiles(1, 4), 512, 0, stream>>>(d, vec_out);
    else gemm_fp8_few_kernel<1, 2, WIDE><<<tiles(1, 2), 512, 0, stream>>>(d, vec_out);
  } else if (d.M <= 32 || tiles(4, 4) < 128) {
    gemm_fp8_few_kernel<2, 4, WIDE><<<tiles(2, 4), 512, 0, stream>>>(d, vec_out);
  } else {
    gemm_fp8_few_kernel<4, 4, WIDE><<<tiles(4, 4), 512, 0, stream>>>(d, vec_out);
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
  if (d->N > 65535 * 64) return ACTH_EINVAL;
  const bool dma = d->K % 16 == 0 && al(d->A, d->lda, 16) && al(d->W, d->ldw, 16) && d->lda < (1 << 22) && d->ldw < (1 << 22) &&
                   d->K <= 128 * 1024 && 256 * d->as_row < (1 << 28) && (d->K + 127) / 128 * d->as_blk < (1 << 28);
  if (dma) {
    const long long t256 = (long long)((d->M + 255) / 256) * ((d->N + 255) / 256);
    const long long t128 = (long long)((d->M + 127) / 128) * ((d->N + 127) / 128);
    // Rounds of the chip: 256 large tiles, or 512 small ones (two blocks a CU), in 1.5 times a small round's time
    // (42 and 27.5 us at K = 2560). 4096 x 2560: 47 against 50 us, 4096 x 5120: 87 against 72, 16384 x 2560: 253 against 276.
    const long long r256 = (t256 + 255) / 256, r128 = (t128 + 511) / 512;
    if (d->M <= 32 || t128 <= 40) {              // 256 x 2560 x 2560: 14.6 against 16.2 us, 512 rows: 27.5 against 16.7

      if (d->out_f32) launch_few<true>(*d, vec_out, stream);
      else launch_few<false>(*d, vec_out, stream);
    } else if (d->out_f32) {
      gemm_fp8_kernel<128, 128, true><<<(unsigned)t128, 512, 0, stream>>>(*d, 16, vec_out);
    } else if (3 * r256 <= 2 * r128) {
      gemm_fp8_kernel<256, 256, false><<<(unsigned)t256, 512, 0, stream>>>(*d, 8, vec_out);
    } else {
      gemm_fp8_kernel<128, 128, false><<<(unsigned)t128, 512, 0, stream>>>(*d, 16, vec_out);
    }
    ACTH_CHECK_LAUNCH();
    return ACTH_OK;
  }
  const dim3 grid((unsigned)((d->M + 63) / 64), (unsigned)((d->N + 63) / 64));
  if (d->out_f32) gemm_fp8_any_kernel<true><<<grid, 256, 0, stream>>>(*d, vec_out);
  else gemm_fp8_any_kernel<false><<<grid, 256, 0, stream>>>(*d, vec_out);
  ACTH_CHECK_LAUNCH();
  return ACTH_OK;
}
