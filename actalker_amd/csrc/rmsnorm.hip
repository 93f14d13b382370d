// Root-mean-square norm with the residual's addition, and 8-bit output with a scale for each 128 columns.
//
//   s = x + res (fp32)      y = s / sqrt(mean(s^2) + eps) * gamma      sum = round(s)
//   8 bits: per row and block of 128 columns  scale = max(max|y|, 2^-100) / 448,  q = e4m3(y / scale)
//
// One pass over the data: a row stays in its lanes' registers between the sum of squares and the output, so each
// input is read once and each output written once. A lane holds chunks of 8 columns (one 16-byte load of 16-bit
// data), 16 neighbouring lanes hold one block of 128, so a block's maximum is four lane exchanges and needs no LDS.
// Bound: HBM bandwidth (32768 x 5120, residual in 16 bits, 8-bit output: 216 us, 5.5 TB/s; 9216 x 1280, fp32 residual: 28 us,
// 5.0 TB/s; on this card a copy of 1 GiB moves 5.1 TB/s, the sum of two into a third 6.0); a few rows: the launch (1 x 2560: 2.9 us).
#include "common.h"

namespace {

constexpr float kTop = 448.0f;                    // the largest e4m3 value
constexpr uint32_t kLeastBits = (127 - 100) << 23;  // 2^-100: the least block maximum

// max |v| over values as integer bits: for non-negative floats the order of the bits is the order of the values,
// and NaN lies above infinity, so a NaN in a block reaches its scale (fmaxf would drop it)
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t umax_(uint32_t a, uint32_t b) { return a > b ? a : b; }

struct Block8 { float inv, scale; };

// scale and its reciprocal from a block's maximum (bits). |y| <= max, so y * inv rounds to at most 448 and the
// conversion never saturates; max = NaN or infinity gives NaN / zero codes, as the division does.
__device__ __forceinline__ Block8 block_scale(uint32_t m) {
  const float amax = __uint_as_float(umax_(m, kLeastBits));
  Block8 b;
  b.scale = amax / kTop;
  b.inv = kTop / amax;
  return b;
}

__device__ __forceinline__ uint2 to_eight8(const float* y, float inv) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// 8 columns of which n are the row's: 16-bit and fp32
template <bool WHOLE>
__device__ __forceinline__ uint4 load8(const bf16_t* p, int n) {
  if (WHOLE) return *reinterpret_cast<const uint4*>(p);
  if (n >= 8) return load16_at(p);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < n) w[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool WHOLE>
__device__ __forceinline__ void load8f(const float* p, int n, float4& a, float4& b) {
  if (WHOLE) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  } else if (n >= 8) {
    const uint4 x = load16_at(p), y = load16_at(p + 4);
    a = make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
    b = make_float4(__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w));
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < n ? p[e] : 0.0f;
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
}

template <bool WHOLE>
__device__ __forceinline__ void store8(bf16_t* p, int n, const float* f) {
  if (WHOLE) {
    *reinterpret_cast<uint4*>(p) = pack8(f);
  } else if (n >= 8) {
    store16_at(p, pack8(f));
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = f2bf(f[e]);
  }
}

template <bool WHOLE>
__device__ __forceinline__ void store8f(float* p, int n, const float* f) {
  if (WHOLE) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else if (n >= 8) {
    store16_at(p, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])));
    store16_at(p + 4, make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])));
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = f[e];
  }
}

// TPR lanes share a row (64: one wave, no barrier; 256: one block), CPL chunks of 8 columns each.
// WHOLE: every chunk has its 8 columns and lies at a multiple of 16 bytes. Otherwise chunks are loaded from any address
// and the row's last one, where it is short, column by column.
template <int TPR, int CPL, bool EIGHT, bool WHOLE>
__global__ __launch_bounds__(256) void rmsnorm_kernel(const ActhRmsNormDesc p) {
  constexpr int ROWS = 256 / TPR;
  const int lane = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool ok = row < p.M;
  const int nch = (p.C + 7) / 8;
  const long long r = ok ? row : 0;
  const bf16_t* xr = (const bf16_t*)p.x + r * p.ldx;

  float s[CPL][8];
  uint4 xv[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int ch = lane + c * TPR;
    xv[c] = make_uint4(0, 0, 0, 0);
    if (ch < nch) xv[c] = load8<WHOLE>(xr + ch * 8, p.C - ch * 8);
  }
  if (p.res && p.res_f32) {
    const float* rr = (const float*)p.res + r * p.ldres;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int ch = lane + c * TPR;
      float4 a = make_float4(0, 0, 0, 0), b = a;
      if (ch < nch) load8f<WHOLE>(rr + ch * 8, p.C - ch * 8, a, b);
      unpack8(xv[c], s[c]);
      s[c][0] += a.x; s[c][1] += a.y; s[c][2] += a.z; s[c][3] += a.w;
      s[c][4] += b.x; s[c][5] += b.y; s[c][6] += b.z; s[c][7] += b.w;
    }
  } else if (p.res) {
    const bf16_t* rr = (const bf16_t*)p.res + r * p.ldres;
    uint4 rv[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int ch = lane + c * TPR;
      rv[c] = make_uint4(0, 0, 0, 0);
      if (ch < nch) rv[c] = load8<WHOLE>(rr + ch * 8, p.C - ch * 8);
    }
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      float t[8];
      unpack8(xv[c], s[c]);
      unpack8(rv[c], t);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] += t[e];
    }
  } else {
#pragma unroll
    for (int c = 0; c < CPL; ++c) unpack8(xv[c], s[c]);
  }

  float rstd = 1.0f;
  if (p.norm) {
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) q = fmaf(s[c][e], s[c][e], q);
    q = wave_sum(q);
    if constexpr (TPR > 64) {
      __shared__ float part[4];
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = q;
      __syncthreads();
      q = (part[0] + part[1]) + (part[2] + part[3]);
    }
    rstd = rsqrtf(q / (float)p.C + p.eps);
  }
  if (!ok) return;                                // after the only barrier; a whole wave leaves together

#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int ch = lane + c * TPR;
    const bool in = ch < nch;
    if (in && p.sum) {
      if (p.res_f32) {
        store8f<WHOLE>((float*)p.sum + row * p.ldsum + ch * 8, p.C - ch * 8, s[c]);
      } else {
        store8<WHOLE>((bf16_t*)p.sum + row * p.ldsum + ch * 8, p.C - ch * 8, s[c]);
      }
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = s[c][e] * rstd;
    if (p.gamma && in) {
      float4 a, b;
      load8f<WHOLE>(p.gamma + ch * 8, p.C - ch * 8, a, b);
      y[0] *= a.x; y[1] *= a.y; y[2] *= a.z; y[3] *= a.w;
      y[4] *= b.x; y[5] *= b.y; y[6] *= b.z; y[7] *= b.w;
    }
    if constexpr (EIGHT) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = umax_(m, in && (WHOLE || ch * 8 + e < p.C) ? mag(y[e]) : 0u);
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) m = umax_(m, (uint32_t)__shfl_xor((int)m, o, 64));
      if (in) {
        const Block8 b = block_scale(m);
        uint8_t* const o = (uint8_t*)p.y + row * p.ldy + ch * 8;
        const uint2 q = to_eight8(y, b.inv);
        if (WHOLE || p.C - ch * 8 >= 8) {
          struct __attribute__((packed, aligned(1))) Any8 { uint32_t v[2]; };
          if (WHOLE) *reinterpret_cast<uint2*>(o) = q;
          else *reinterpret_cast<Any8*>(o) = Any8{{q.x, q.y}};
        } else {
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (ch * 8 + e < p.C) o[e] = (uint8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
        }
        if ((ch & 15) == 0) p.scale[row * p.scale_row + (ch >> 4) * p.scale_blk] = b.scale;
      }
    } else if (in) {
      store8<WHOLE>((bf16_t*)p.y + row * p.ldy + ch * 8, p.C - ch * 8, y);
    }
  }
}

// Rows too wide for a block's registers: a block of 256 walks its row twice, one column a lane (the second read comes from
// L2). A wave takes a block of 128 columns at a time, so a block's maximum stays inside the wave. Columns are summed
// in a fixed order. A sum or output that lies on an input is written only by the lane that has just read it.
template <bool EIGHT>
__global__ __launch_bounds__(256) void rmsnorm_any_kernel(const ActhRmsNormDesc p) {
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bf16_t* xr = (const bf16_t*)p.x + row * p.ldx;
  auto load = [&](int c) {
    float v = bf2f(xr[c]);
    if (p.res) v += p.res_f32 ? ((const float*)p.res)[row * p.ldres + c] : bf2f(((const bf16_t*)p.res)[row * p.ldres + c]);
    return v;
  };
  float rstd = 1.0f;
  if (p.norm) {
    float q = 0.0f;
    for (int c = threadIdx.x; c < p.C; c += 256) {
      const float v = load(c);
      q = fmaf(v, v, q);
    }
    q = wave_sum(q);
    __shared__ float part[4];
    if (lane == 0) part[wave] = q;
    __syncthreads();
    q = (part[0] + part[1]) + (part[2] + part[3]);
    rstd = rsqrtf(q / (float)p.C + p.eps);
  }
  for (int c0 = wave * 128; c0 < p.C; c0 += 512) {
    float y[2];
    uint32_t m = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = c0 + h * 64 + lane;
      y[h] = 0.0f;
      if (c < p.C) {
        const float v = load(c);
        y[h] = v * rstd;
        if (p.gamma) y[h] *= p.gamma[c];
        m = umax_(m, mag(y[h]));
        if (p.sum) {
          if (p.res_f32) ((float*)p.sum)[row * p.ldsum + c] = v;
          else ((bf16_t*)p.sum)[row * p.ldsum + c] = f2bf(v);
        }
        if constexpr (!EIGHT) ((bf16_t*)p.y)[row * p.ldy + c] = f2bf(y[h]);
      }
    }
    if constexpr (EIGHT) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) m = umax_(m, (uint32_t)__shfl_xor((int)m, o, 64));
      const Block8 b = block_scale(m);
      const int two = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * b.inv, y[1] * b.inv, 0, false);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + h * 64 + lane;
        if (c < p.C) ((uint8_t*)p.y)[row * p.ldy + c] = (uint8_t)(two >> (8 * h));
      }
      if (lane == 0) p.scale[row * p.scale_row + (c0 >> 7) * p.scale_blk] = b.scale;
    }
  }
}

template <int TPR, int CPL>
void launch(const ActhRmsNormDesc& d, bool whole, hipStream_t stream) {
  const unsigned grid = (unsigned)((d.M + 256 / TPR - 1) / (256 / TPR));
  if (d.eight && whole) rmsnorm_kernel<TPR, CPL, true, true><<<grid, 256, 0, stream>>>(d);
  else if (d.eight) rmsnorm_kernel<TPR, CPL, true, false><<<grid, 256, 0, stream>>>(d);
  else if (whole) rmsnorm_kernel<TPR, CPL, false, true><<<grid, 256, 0, stream>>>(d);
  else rmsnorm_kernel<TPR, CPL, false, false><<<grid, 256, 0, stream>>>(d);
}

bool aligned(const void* p, long long ld_bytes, int to) {
  return !p || (((uintptr_t)p | (uintptr_t)ld_bytes) % to) == 0;
}

}  // namespace

extern "C" int acth_rmsnorm(const ActhRmsNormDesc* d, hipStream_t stream) {
  if (!d || d->M < 0) return ACTH_EINVAL;
  if (d->M == 0) return ACTH_OK;
  if (d->C < 1 || d->C > (1 << 30) || !d->x || !d->y || (d->eight && !d->scale)) return ACTH_EINVAL;
  if (d->M > 1 && (d->ldx < d->C || d->ldy < d->C || (d->res && d->ldres < d->C) || (d->sum && d->ldsum < d->C)))
    return ACTH_EINVAL;
  const int rs = d->res_f32 ? 4 : 2;
  const bool whole = d->C % 8 == 0 && aligned(d->x, d->ldx * 2, 16) && aligned(d->res, d->ldres * rs, 16) &&
                     aligned(d->sum, d->ldsum * rs, 16) && aligned(d->gamma, 0, 16) &&
                     aligned(d->y, d->ldy * (d->eight ? 1 : 2), d->eight ? 8 : 16);
  const int nch = (d->C + 7) / 8;
  constexpr int ROWS = (1 << 24) - 8;              // a launch holds less than 2^32 lanes, a row takes up to 256
  if (d->M > ROWS) {
    for (long long m = 0; m < d->M; m += ROWS) {
      ActhRmsNormDesc s = *d;
      s.M = d->M - m < ROWS ? (int)(d->M - m) : ROWS;
      s.x = (const bf16_t*)d->x + m * d->ldx;
      if (d->res) s.res = (const char*)d->res + m * d->ldres * rs;
      if (d->sum) s.sum = (char*)d->sum + m * d->ldsum * rs;
      s.y = (char*)d->y + m * d->ldy * (d->eight ? 1 : 2);
      if (d->scale) s.scale = d->scale + m * d->scale_row;
      const int rc = acth_rmsnorm(&s, stream);
      if (rc) return rc;
    }
    return ACTH_OK;
  }
  // A wave a row up to 2048 columns, a block above: 32768 x 1280 54 against 69 us, 2048 x 2560 9.1 against 8.6,
  // 32768 x 5120 225 against 219, 64 x 5120 8.9 against 4.7 (8-bit output, residual in 16 bits).
  if (nch <= 64) launch<64, 1>(*d, whole, stream);
  else if (nch <= 128) launch<64, 2>(*d, whole, stream);
  else if (nch <= 192) launch<64, 3>(*d, whole, stream);
  else if (nch <= 256) launch<64, 4>(*d, whole, stream);
  else if (nch <= 512) launch<256, 2>(*d, whole, stream);
  else if (nch <= 768) launch<256, 3>(*d, whole, stream);
  else if (nch <= 1024) launch<256, 4>(*d, whole, stream);
  else if (nch <= 2048) launch<256, 8>(*d, whole, stream);
  else if (d->eight) rmsnorm_any_kernel<true><<<d->M, 256, 0, stream>>>(*d);
  else rmsnorm_any_kernel<false><<<d->M, 256, 0, stream>>>(*d);
  ACTH_CHECK_LAUNCH();
  return ACTH_OK;
}
