// The sequence part of a gated state-space layer, for prompts and for single tokens: the short causal convolution and
// the selective scan, over ragged sequences whose states are kept between calls.
//
//   convolution   y[t] = silu(bias + sum_j w[j] x[t - W + 1 + j])          rows before the sequence: the kept W - 1 inputs
//   scan          dt = softplus(delta + bias),  h = exp(dt A) h + dt u B,  y = (C h + D u) silu(z)
//
// Sequences are row ranges [starts[i], starts[i+1]) of one token-major tensor; `starts` lives on the device, so the
// host never learns the lengths. Everything read from it is clamped to [0, T], and a slot outside [0, nslots) marks a
// padding sequence whose rows are left alone, so no content of either can lead an access out of its tensor.
#include <type_traits>

#include "common.h"

namespace {

// ------------------------------------------------------------------------------------------------ sequences
struct Seq { int i, s, e, slot; };                 // sequence i holds rows [s, e); slot -1: none or padding

template <class P>
__device__ __forceinline__ int seq_start(const P& p, int i) {
  if (!p.starts) return (int)((long long)i * (p.T / p.nseq));
  const int v = p.starts[i];
  return v < 0 ? 0 : v > p.T ? p.T : v;
}

template <class P>
__device__ __forceinline__ int seq_slot(const P& p, int i) {
  const int v = p.slots ? p.slots[i] : i;
  return v >= 0 && v < p.nslots ? v : -1;
}

template <class P>
__device__ __forceinline__ Seq seq_of(const P& p, int i) {
  Seq q;
  q.i = i;
  q.s = i < p.nseq ? seq_start(p, i) : p.T;
  q.e = i < p.nseq ? seq_start(p, i + 1) : p.T;
  q.slot = i < p.nseq ? seq_slot(p, i) : -1;
  return q;
}

// the sequence that holds row t: the last one that starts at or before t (empty ones in front of it start there too);
// i = -1 where the first one starts behind t
template <class P>
__device__ __forceinline__ Seq seq_find(const P& p, int t) {
  if (!p.starts) return seq_of(p, t / (p.T / p.nseq));
  int lo = 0, hi = p.nseq;                         // first index in [0, nseq) whose start lies behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (seq_start(p, mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo == 0) {
    Seq q;
    q.i = -1; q.s = 0; q.e = seq_start(p, 0); q.slot = -1;
    return q;
  }
  return seq_of(p, lo - 1);
}

template <class P>
__device__ __forceinline__ bool seq_kept(const P& p, const Seq& q) {        // does it go on from a kept state?
  return p.state && q.slot >= 0 && !(p.fresh && p.fresh[q.i]);
}

// the sequence behind q that may hold row t or a later one: not one by one over empty ones, of which a padded batch has
// many in one place (a search from the front, which offsets out of order cannot lead back)
template <class P>
__device__ __forceinline__ Seq seq_next(const P& p, const Seq& q, int t) {
  Seq n = seq_of(p, q.i + 1);
  if (p.starts && n.i < p.nseq && n.e <= t) {
    const Seq f = seq_find(p, t);
    if (f.i > n.i) n = f;
  }
  return n;
}

constexpr float kLog2e = 1.4426950408889634f;

// x / (1 + exp(-x)) with the one-step reciprocal, for 16-bit outputs. The exponential and the reciprocal are off by 2
// roundings of 2^-24 each, the sum and the product by one; the exponent's own roundings make the exponential off by 1.3 |x|
// more. Where x > 0 that weighs e / (1 + e) < exp(-x), less than half a rounding; where x < 0 it weighs up to 1: within
// 6 + 1.3 |x| roundings, 2^-19 at x = -20.
__device__ __forceinline__ float silu16(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// ------------------------------------------------------------------------------------------------ convolution
// VEC channels a lane (8: one 16-byte load a row, from any address; 1: fewer than 8 channels), a wave 64 x VEC channels of CT rows. The
// rows of a tile are loaded before the first is used; the W - 1 rows in front of it are read again (3 beside 16, from L2).
// The tile that holds a sequence's first row also takes the rows that reach back into the kept inputs and writes the
// new ones, so one lane both reads and writes each kept value. Bound: HBM bandwidth (32768 x 5120 x 4 taps, 24 sequences:
// 154 us, 4.4 TB/s; 8 or 32 rows a tile: 168, 154; channels that fill no 8: 190).

template <int VEC>
__device__ __forceinline__ void load_c(const bf16_t* p, float* f) {
  if constexpr (VEC == 8) unpack8(load16_at(p), f);
  else f[0] = bf2f(*p);
}

// the channels from `e0` on: the lane of a row's end, where that is short, lies back over its neighbour's channels and
// leaves those to it
template <int VEC>
__device__ __forceinline__ void store_c(bf16_t* p, const float* f, int e0) {
  if constexpr (VEC == 8) {
    if (e0 == 0) {
      store16_at(p, pack8(f));
    } else {
#pragma unroll
      for (int e = 1; e < 8; ++e)
        if (e >= e0) p[e] = f2bf(f[e]);
    }
  } else {
    *p = f2bf(f[0]);
  }
}

template <int VEC> struct Raw { typedef bf16_t type; };
template <> struct Raw<8> { typedef uint4 type; };

template <int VEC>
__device__ __forceinline__ typename Raw<VEC>::type load_raw(const bf16_t* p) {
  if constexpr (VEC == 8) return load16_at(p);
  else return *p;
}

template <int VEC>
__device__ __forceinline__ void from_raw(const typename Raw<VEC>::type v, float* f) {
  if constexpr (VEC == 8) unpack8(v, f);
  else f[0] = bf2f(v);
}

template <int VEC, int W>
struct ConvLane {
  float w[W][VEC], b[VEC];
  int silu;
  __device__ __forceinline__ void init(const ActhCausalConvDesc& p, int d) {
    silu = p.silu;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      b[v] = p.bias ? p.bias[d + v] : 0.0f;
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][v] = p.w[(long long)(d + v) * W + j];
    }
  }
  // win: the W - 1 inputs before x, oldest first. Two evaluations, both within the fp32 error of the formula, so that their
  // 16-bit results differ only where the value lies that near a tie. Against 64 bits the fused one (sums by multiply-adds, quick
  // quotient) falls on the other side of a tie for 2.8e-5 of bf16 values and 1.8e-4 of fp16 ones, the stepwise one (each
  // product and sum rounded, accurate exponential and quotient) for 4.0e-5 and 2.4e-4. Prompts take the fused one (32768 x 5120:
  // 154 against 212 us). Steps take the stepwise one, although it costs 1.7 us at 512 x 5120: it is what the formula gives in
  // fp32 operation by operation, as a program outside these kernels evaluates it, and a state of 32 bits keeps for good what one
  // 16-bit rounding of its input does (7e-4 of its size at worst in 40 million states; 5e-7 this way).
  template <bool STEPWISE>
  __device__ __forceinline__ void out(const float (*win)[VEC], const float* x, float* y) const {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      if constexpr (STEPWISE) {
#pragma clang fp contract(off)
        float a = w[0][v] * win[0][v];
#pragma unroll
        for (int j = 1; j < W - 1; ++j) a = a + w[j][v] * win[j][v];
        a = a + w[W - 1][v] * x[v];
        a = a + b[v];
        y[v] = silu ? a / (1.0f + expf(-a)) : a;
      } else {
        float a = b[v];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) a = fmaf(w[j][v], win[j][v], a);
        a = fmaf(w[W - 1][v], x[v], a);
        y[v] = silu ? silu16(a) : a;
      }
    }
  }
  static __device__ __forceinline__ void shift(float (*win)[VEC], const float* x) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
#pragma unroll
      for (int j = 0; j + 1 < W - 1; ++j) win[j][v] = win[j + 1][v];
      win[W - 2][v] = x[v];
    }
  }
};

template <int VEC, int W, int CT>
__global__ __launch_bounds__(64) void causal_conv_kernel(const ActhCausalConvDesc p) {
  const int t0 = blockIdx.x * CT, t1 = min(t0 + CT, p.T);
  const int d_ = (blockIdx.y * 64 + threadIdx.x) * VEC;
  if (d_ >= p.D) return;
  const int d = min(d_, p.D - VEC), e0 = d_ - d;
  ConvLane<VEC, W> c;
  c.init(p, d);
  const bf16_t* x = (const bf16_t*)p.x + d;
  bf16_t* y = (bf16_t*)p.y + d;
  bf16_t* state = (bf16_t*)p.state + d;
  Seq q = seq_find(p, t0);
  float win[W - 1][VEC], xv[VEC], yv[VEC];

  if (q.i >= 0 && t0 - q.s >= W - 1 && q.e >= t1 && t1 - t0 == CT) {           // all rows inside one sequence
    if (p.slots && q.slot < 0) return;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) load_c<VEC>(x + (long long)(t0 - (W - 1) + j) * p.ldx, win[j]);
#pragma unroll
    for (int k = 0; k < CT; ++k) {
      load_c<VEC>(x + (long long)(t0 + k) * p.ldx, xv);
      c.template out<false>(win, xv, yv);
      store_c<VEC>(y + (long long)(t0 + k) * p.ldy, yv, e0);
      c.shift(win, xv);
    }
    return;
  }

  int t = t0;
  while (t < t1) {
    if (q.i < 0 || q.i >= p.nseq || q.e <= t) {                  // rows that no sequence holds, or an empty sequence
      if (q.i >= p.nseq) return;
      if (q.i < 0) t = max(t, q.e);
      q = seq_next(p, q, t);
      if (q.i < p.nseq && q.s > t) t = q.s;
      continue;
    }
    const bool has = !p.slots || q.slot >= 0;
    const bool own = q.s >= t0;                                  // this tile holds the sequence's first row
    const bool kept = seq_kept(p, q);
    bf16_t* st = state + (long long)(q.slot < 0 ? 0 : q.slot) * p.ld_slot;
    float init[W - 1][VEC];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) init[j][v] = 0.0f;
      if (own && kept) load_c<VEC>(st + (long long)j * p.D, init[j]);
    }
    // its first row here: rows that reach back before the sequence belong to the tile that holds its first row
    int a = own ? q.s : max(t, q.s + W - 1);
    int b = min(q.e, t1);
    if (own) b = min(q.e, max(t1, q.s + W - 1));
    if (has && a < b) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        if (own) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) win[j][v] = init[j][v];
        } else {
          load_c<VEC>(x + (long long)(a - (W - 1) + j) * p.ldx, win[j]);
        }
      }
      for (int r = a; r < b; ++r) {
        load_c<VEC>(x + (long long)r * p.ldx, xv);
        c.template out<false>(win, xv, yv);
        store_c<VEC>(y + (long long)r * p.ldy, yv, e0);
        c.shift(win, xv);
      }
    }
    if (own && p.state && q.slot >= 0 && q.e > q.s) {
      const int len = q.e - q.s;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        const int r = len - (W - 1) + j;                         // row of the sequence, or a kept input before it
        float nv[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) nv[v] = 0.0f;
        if (r >= 0) {
          load_c<VEC>(x + (long long)(q.s + r) * p.ldx, nv);
        } else {
#pragma unroll
          for (int k = 0; k < W - 1; ++k)
            if (k == r + W - 1) {
#pragma unroll
              for (int v = 0; v < VEC; ++v) nv[v] = init[k][v];
            }
        }
        store_c<VEC>(st + (long long)j * p.D, nv, e0);
      }
    }
    t = max(t, q.e);
    q = seq_next(p, q, t);
    if (q.i < p.nseq && q.s > t) t = q.s;
  }
}

// sequences a lane, once there are blocks enough: 1, 2, 4, 8 of them in a graph 512 x 5120 16.7, 12.2, 13.0, 14.4 us, 2048 x
// 5120 54, 36.9, 33.3, 38.0, 300 x 5120 12.2, 9.7, 9.3, 13.6; 128 x 5120 7.3, 6.1, 8.2, 12.7
constexpr int CSTEP = 4;

// One row a sequence: a lane takes VEC channels of SEQS sequences, whose loads are all under way before the first is
// used, so that the weights are read once for them. Bound: the kept inputs' bytes; few rows: the launch.
template <int VEC, int W, int SEQS>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(const ActhCausalConvDesc p) {
  const int nb = (p.D + 256 * VEC - 1) / (256 * VEC);      // channel blocks, the fastest
  const int bs = blockIdx.x / nb, d_ = ((blockIdx.x - bs * nb) * 256 + threadIdx.x) * VEC;
  if (d_ >= p.D) return;
  const int d = min(d_, p.D - VEC), e0 = d_ - d;
  const int r0 = bs * SEQS;
  typedef typename Raw<VEC>::type raw_t;
  raw_t xr[SEQS], wr[SEQS][W - 1];
  int slot[SEQS];
  bool kept[SEQS], live[SEQS];
#pragma unroll
  for (int k = 0; k < SEQS; ++k) {
    const int r = min(r0 + k, p.T - 1);
    const Seq q = seq_of(p, r);
    live[k] = r0 + k < p.T && (!p.slots || q.slot >= 0);
    slot[k] = q.slot;
    kept[k] = seq_kept(p, q);
    xr[k] = load_raw<VEC>((const bf16_t*)p.x + (long long)r * p.ldx + d);
    const bf16_t* st = (const bf16_t*)p.state + (q.slot < 0 ? 0 : q.slot) * p.ld_slot + d;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      wr[k][j] = raw_t{};
      if (kept[k]) wr[k][j] = load_raw<VEC>(st + (long long)j * p.D);
    }
  }
  ConvLane<VEC, W> c;
  c.init(p, d);
#pragma unroll
  for (int k = 0; k < SEQS; ++k) {
    if (!live[k]) continue;
    float win[W - 1][VEC], xv[VEC], yv[VEC];
    from_raw<VEC>(xr[k], xv);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) from_raw<VEC>(wr[k][j], win[j]);
    c.template out<true>(win, xv, yv);
    store_c<VEC>((bf16_t*)p.y + (long long)(r0 + k) * p.ldy + d, yv, e0);
    if (p.state && slot[k] >= 0) {                 // the kept inputs move up by one
      c.shift(win, xv);
      bf16_t* st = (bf16_t*)p.state + slot[k] * p.ld_slot + d;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) store_c<VEC>(st + (long long)j * p.D, win[j], e0);
    }
  }
}

// A launch holds less than 2^32 lanes: rows that blocks of 256 lanes, `per_row` of them a row, may take in one
constexpr int LAUNCH = 1 << 24;
int launch_rows(long long per_row) { return (int)((LAUNCH - 1) / per_row) & ~7; }

// rows [t0, t0 + n) of a step, which is one sequence a row
template <class P>
P step_rows(P d, int t0, int n) {
  d.T = d.nseq = n;
  if (d.fresh) d.fresh += t0;
  if (d.slots) {
    d.slots += t0;
  } else if (d.state) {
    d.state = (decltype(d.state))((char*)d.state + t0 * d.ld_slot * (std::is_same<P, ActhSsmScanDesc>::value ? 4 : 2));
    d.nslots -= t0;
  }
  return d;
}

template <int VEC, int W>
void launch_conv(const ActhCausalConvDesc& d, hipStream_t stream) {
  if (!d.starts && d.nseq == d.T) {
    const unsigned bx = (unsigned)((d.D + 256 * VEC - 1) / (256 * VEC));
    const int rows = launch_rows(bx);
    for (int t0 = 0; t0 < d.T; t0 += rows) {
      ActhCausalConvDesc s = step_rows(d, t0, d.T - t0 < rows ? d.T - t0 : rows);
      s.x = (const bf16_t*)d.x + t0 * d.ldx;
      s.y = (bf16_t*)d.y + t0 * d.ldy;
      if ((long long)bx * s.T >= 1024) causal_conv_step_kernel<VEC, W, CSTEP><<<(unsigned)((s.T + CSTEP - 1) / CSTEP) * bx, 256, 0, stream>>>(s);
      else causal_conv_step_kernel<VEC, W, 1><<<(unsigned)s.T * bx, 256, 0, stream>>>(s);
    }
  } else {
    const unsigned by = (unsigned)((d.D + 64 * VEC - 1) / (64 * VEC));
    const auto tiles = [&](int rows) { return dim3((unsigned)((d.T + rows - 1) / rows), by); };
    // Tiles of 16 rows that leave SIMDs idle (there are 1024) are cut: 4, 8, 16 rows, a call in a graph: 300 x 640 6.2, 7.0,
    // 10.1 us, 1000 x 1306 7.8, 9.2, 12.0; 1000 x 5120 11.8, 10.1, 11.2, 4000 x 2560 16.5, 14.2, 16.6; 8000 x 2560 24.0, 22.1, 20.2.
    const long long waves = (long long)tiles(16).x * by;
    if (waves < 512) causal_conv_kernel<VEC, W, 4><<<tiles(4), 64, 0, stream>>>(d);
    else if (waves < 2048) causal_conv_kernel<VEC, W, 8><<<tiles(8), 64, 0, stream>>>(d);
    else causal_conv_kernel<VEC, W, 16><<<tiles(16), 64, 0, stream>>>(d);
  }
}

// ------------------------------------------------------------------------------------------------ scan

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1]. With w = 1 + e rounded and c = e - (w - 1) what the
// rounding lost (at most 2^-24), log1p(e) = log(w) + c / w + ..., and c stands for c / w: they differ by at most
// 2^-24 e / (1 + e), one rounding of the result. So small e keep their digits, which log(1 + e) alone would lose, for 7
// operations and two of the slow ones.
__device__ __forceinline__ float softplus16(float x) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
  const float w = 1.0f + e;
  const float c = e - (w - 1.0f);
  return fmaxf(x, 0.0f) + fmaf(__builtin_amdgcn_logf(w), 0.69314718055994531f, c);   // NaN passes through e
}

__device__ __forceinline__ float load_any(const void* p, long long i, int f32) {
  return f32 ? ((const float*)p)[i] : bf2f(((const bf16_t*)p)[i]);
}

// A long sequence is cut into chunks of at most `len` rows, so that few rows fill the chip as well:
//   pass 1 (LOCAL)   every chunk but a sequence's last, the first one from the sequence's start state and the others from
//                    zero: its end state, and the sum of its time steps, which gives its decay exp(A sum dt);
//   carry            the true states at the chunks' starts, one after the other, a lane per channel and state;
//   pass 2 (FINAL)   every chunk from its start state: outputs, and the sequence's new state.
// A sequence of one chunk takes pass 2 alone. Chunk k of sequence i is found on the device from the offsets. The start
// states of a sequence's chunks lie in consecutive places of the workspace, the first one's among them: pass 2 writes
// the kept states, so nothing may read them there any more.
struct Chunks {
  int len, n, places;                              // rows a chunk; bounds of the chunks and of the workspace's places
  float* h;                                        // (places, D, N): end states at the next chunk's place, then start states
  float* s;                                        // (places, D): sums of the time steps of the chunk before
  int* kind;                                       // (places): 0 a start state as it is, 1 decays what comes before it
};

struct Chunk { int i, slot, r0, r1, j, c, place; };     // chunk j of the c of sequence i, rows [r0, r1); i = -1: none

// Lane by lane over the sequences, 64 at a time: prefix sums of their chunks, and of those of sequences of several.
// idx < 0: the sums over all sequences (r0 chunks, place places).
template <class P>
__device__ __forceinline__ Chunk chunk_find(const P& p, const Chunks& ck, int idx) {
  Chunk k{};
  k.i = -1;
  if (!p.starts) {
    const int L = p.T / p.nseq, c = (L + ck.len - 1) / ck.len;
    if (idx < 0) {
      k.r0 = c * p.nseq;
      k.place = c > 1 ? k.r0 : 0;
      return k;
    }
    if (idx >= c * p.nseq) return k;
    const int i = idx / c;
    k.slot = seq_slot(p, i);
    if (p.slots && k.slot < 0) return k;
    k.i = i;
    k.j = idx - i * c;
    k.c = c;
    k.place = c > 1 ? i * c : 0;
    k.r0 = i * L + k.j * ck.len;
    k.r1 = min(k.r0 + ck.len, i * L + L);
    return k;
  }
  const int lane = threadIdx.x & 63;
  int before = 0, multi = 0;
  for (int i0 = 0; i0 < p.nseq; i0 += 64) {
    const int i = i0 + lane;
    int s = 0, e = 0, slot = -1, c = 0, len = ck.len;
    if (i < p.nseq) {
      s = seq_start(p, i);
      e = seq_start(p, i + 1);
      slot = seq_slot(p, i);
      if (e > s && (!p.slots || slot >= 0)) {      // about equal chunks: a short last one would leave its place idle
        c = (e - s + ck.len - 1) / ck.len;
        len = ((e - s + c - 1) / c + 7) & ~7;
        c = (e - s + len - 1) / len;
      }
    }
    const int m = c > 1 ? c : 0;
    int x = c, y = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int vx = __shfl_up(x, o, 64), vy = __shfl_up(y, o, 64);
      if (lane >= o) { x += vx; y += vy; }
    }
    const int total = __shfl(x, 63, 64);
    if (idx >= 0 && idx - before < total) {
      const int at = __ffsll((unsigned long long)__ballot(x > idx - before)) - 1;
      const int c0 = before + __shfl(x - c, at, 64);
      k.i = i0 + at;
      k.c = __shfl(c, at, 64);
      k.j = idx - c0;
      k.place = multi + __shfl(y - m, at, 64);
      k.slot = __shfl(slot, at, 64);
      len = __shfl(len, at, 64);
      k.r0 = __shfl(s, at, 64) + k.j * len;
      k.r1 = min(k.r0 + len, __shfl(e, at, 64));
      if (k.c > 1 && k.place + k.c > ck.places) k.i = -1;      // offsets that overlap: not more than there is room for
      return k;
    }
    before += total;
    multi += __shfl(y, 63, 64);
  }
  k.r0 = before;
  k.place = multi;
  return k;
}

constexpr int TT = 8;                             // rows of a tile in LDS

// f[i] for i < 8 without addressing registers; 0 behind
__device__ __forceinline__ float select8(const float* f, int i) {
  float v = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) v = i == e ? f[e] : v;
  return v;
}

template <int VEC>
__device__ __forceinline__ uint4 load16_v(const void* p) {
  if constexpr (VEC == 2) return *reinterpret_cast<const uint4*>(p);
  else return load16_at(p);
}

// A wave takes CB channels of a chunk: SPL states a lane, LPC lanes a channel, CPT channels a lane. A tile's time steps
// (softplus done once, by the staging lane) and inputs dt u sit in LDS as pairs beside the rows of B and C; the output
// takes the place of the pair that its own lane has just read. The next tile's rows are loaded while this one is
// walked. One wave a block, so no barrier waits for another wave.
// Channel c of a row lies at place (c % 8)(CB / 8) + c / 8, and rows are CB bytes further apart than they are long:
// the staging lanes, which hold 8 neighbouring channels each, then write neighbouring places (laid out by channel they
// met in 4 banks, 16 at a time), and the walking lanes read one place each.
// Bound: the vector units, a row, channel and state taking one exponential (8 clocks a wave) and four operations (4 each):
// 8192 x 2560 x 16 states 51 us in pass 2 and 43 in pass 1 if nothing else were done; 101 and 80 measured, the rest being
// the softplus, gate and conversions of the staging lanes and the waves' waits (the units are 75 - 79 % busy).
// VEC: 2 pieces of 8 channels at multiples of 16 bytes, 1 at any address, 0 groups of fewer than 8 channels
template <int SPL, int LPC, int CPT, bool LOCAL, int VEC>
__global__ __launch_bounds__(64, 3) void ssm_scan_kernel(const ActhSsmScanDesc p, const Chunks ck) {
  constexpr int CL = 64 / LPC;                     // channels a wave holds at once
  constexpr int CB = CL * CPT;
  constexpr int NS = SPL * LPC;
  constexpr int C8 = CB / 8;                       // 8-channel pieces a row
  constexpr int E8 = C8 * TT > 64 ? C8 * TT / 64 : 1;     // pieces a lane
  constexpr int NB = TT * NS / 64;                 // values of B (and C) a lane
  constexpr int PITCH = CB + C8;
  __shared__ __align__(16) float2 sx[TT][PITCH];
  __shared__ __align__(16) float sb[TT][NS], sc[LOCAL ? 1 : TT][NS];
  __shared__ __align__(16) float s_bias[CB], s_skip[CB];

  const int lane = threadIdx.x;
  const Chunk q = chunk_find(p, ck, blockIdx.x);
  if (q.i < 0 || (LOCAL && q.j + 1 >= q.c)) return;
  const int c0 = q.r0, c1 = q.r1;
  const int dg = p.D / p.G, nb = (dg + CB - 1) / CB;
  const int g = blockIdx.y / nb;
  const int d0 = g * dg + (blockIdx.y - g * nb) * CB, d1 = min(d0 + CB, (g + 1) * dg);

  // ---- loads of a tile, held until the tile before it is done. A lane's places move down TT rows a tile. Rows behind
  // the chunk are not loaded; a piece that the group's end cuts is loaded from 8 channels before the end and moved down by
  // `back`: what lies behind the end is never walked or never stored. States behind the last one keep zeros.
  uint4 pu[E8], pd[E8][2];
  uint32_t pb[NB], pc[NB];                         // raw: a conversion here would wait for its load
  const int dsz = p.delta_f32 ? 4 : 2, bsz = p.bc_f32 ? 4 : 2;
  const int fr = lane / C8, fd = min(d0 + lane % C8 * 8, d1 - 8);      // (VEC: a group has 8 channels or more)
  const int back = min(d0 + lane % C8 * 8 - fd, 7);
  const bool cut = VEC == 1 && ((d1 - d0) & 7) != 0;      // the same for the wave: most have no such piece
  const int gr = lane / NS, gn = lane % NS;
  const bf16_t* at_u = (const bf16_t*)p.u + (long long)(c0 + fr) * p.ldu + fd;
  const char* at_d = (const char*)p.delta + ((long long)(c0 + fr) * p.ld_delta + fd) * dsz;
  const char* at_b = (const char*)p.B + ((long long)(c0 + gr) * p.ldb + g * p.N + gn) * bsz;
  const char* at_c = (const char*)p.C + ((long long)(c0 + gr) * p.ldc + g * p.N + gn) * bsz;
#pragma unroll
  for (int k = 0; k < NB; ++k) pb[k] = pc[k] = 0;
  auto fetch = [&](int b0) {
    const int left = c1 - b0;
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < E8; ++k) {
        const int r = fr + 64 / C8 * k;
        if (r < TT && r < left) {
          pu[k] = load16_v<VEC>(at_u + (long long)(64 / C8 * k) * p.ldu);
          const char* f = at_d + (long long)(64 / C8 * k) * p.ld_delta * dsz;
          pd[k][0] = load16_v<VEC>(f);
          if (p.delta_f32) pd[k][1] = load16_v<VEC>(f + 16);
        }
      }
      at_u += (long long)TT * p.ldu;
      at_d += (long long)TT * p.ld_delta * dsz;
    }
    if (gn < p.N) {
#pragma unroll
      for (int k = 0; k < NB; ++k)
        if (gr + 64 / NS * k < left) {
          const long long ob = (long long)(64 / NS * k) * p.ldb * bsz, oc = (long long)(64 / NS * k) * p.ldc * bsz;
          if (p.bc_f32) {
            pb[k] = *reinterpret_cast<const uint32_t*>(at_b + ob);
            if (!LOCAL) pc[k] = *reinterpret_cast<const uint32_t*>(at_c + oc);
          } else {
            pb[k] = *reinterpret_cast<const bf16_t*>(at_b + ob);
            if (!LOCAL) pc[k] = *reinterpret_cast<const bf16_t*>(at_c + oc);
          }
        }
    }
    at_b += (long long)TT * p.ldb * bsz;
    at_c += (long long)TT * p.ldc * bsz;
  };
  fetch(c0);
  for (int c = lane; c < CB; c += 64) {
    s_bias[c] = p.delta_bias && d0 + c < d1 ? p.delta_bias[d0 + c] : 0.0f;
    s_skip[c] = p.Dskip && d0 + c < d1 ? p.Dskip[d0 + c] : 0.0f;
  }

  const int part = lane % LPC;
  auto place = [&](int j) { return lane / LPC + CL * j; };
  auto channel = [&](int j) { return d0 + place(j) % C8 * 8 + place(j) / C8; };
  float A[CPT][SPL], h[CPT][SPL], sum[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    sum[j] = 0.0f;
    const int d = channel(j);
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      const int n = part * SPL + s;
      const float a = p.A[(long long)min(d, d1 - 1) * p.N + min(n, p.N - 1)] * kLog2e;     // loads without branches
      A[j][s] = n < p.N ? a : 0.0f;
      h[j][s] = 0.0f;
    }
  }
  auto load_h = [&](const float* from) {           // from: (D, N)
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
      for (int s = 0; s < SPL; ++s) h[j][s] = from[(long long)min(channel(j), d1 - 1) * p.N + min(part * SPL + s, p.N - 1)];
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
      for (int s = 0; s < SPL; ++s)
        if (part * SPL + s >= p.N) h[j][s] = 0.0f;
  };
  // every load of a state or of A ends before the walk: left under way, it would make the walk's first use of a state
  // wait for all loads, the next tile's among them
  auto pin = [&]() {
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
      for (int s = 0; s < SPL; ++s) asm volatile("" : "+v"(h[j][s]), "+v"(A[j][s]));
  };
  auto store_h = [&](float* to) {
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
      for (int s = 0; s < SPL; ++s) {
        const int d = channel(j), n = part * SPL + s;
        if (d < d1 && n < p.N) to[(long long)d * p.N + n] = h[j][s];
      }
  };
  const long long dn = (long long)p.D * p.N;
  float* const state = p.state + (p.state ? q.slot * p.ld_slot : 0);
  if (!LOCAL && q.c > 1) load_h(ck.h + (q.place + q.j) * dn);
  else if (q.j == 0 && p.state && !(p.fresh && p.fresh[q.i])) load_h(state);
  pin();
  if (LOCAL && q.j == 0) store_h(ck.h + q.place * dn);

  __syncthreads();
  for (int b0 = c0; b0 < c1; b0 += TT) {
    const int b1 = min(b0 + TT, c1);
    // ---- the tile into LDS
    uint4 u[E8], z[E8];
#pragma unroll
    for (int k = 0; k < E8; ++k) {
      const int piece = lane + 64 * k, r = piece / C8, o = piece % C8, d = d0 + o * 8;
      const long long row = b0 + r;
      const bool in = r < TT && b0 + r < b1;
      float uf[8], dl[8];
      if constexpr (VEC) {
        u[k] = pu[k];
        if (cut) u[k] = down16(u[k], back);
        if (p.delta_f32) {
          dl[0] = __uint_as_float(pd[k][0].x); dl[1] = __uint_as_float(pd[k][0].y);
          dl[2] = __uint_as_float(pd[k][0].z); dl[3] = __uint_as_float(pd[k][0].w);
          dl[4] = __uint_as_float(pd[k][1].x); dl[5] = __uint_as_float(pd[k][1].y);
          dl[6] = __uint_as_float(pd[k][1].z); dl[7] = __uint_as_float(pd[k][1].w);
          if (cut) {
#pragma unroll
            for (int e = 0; e < 8; ++e) dl[e] = select8(dl, e + back);
          }
        } else {
          uint4 w = pd[k][0];
          if (cut) w = down16(w, back);
          unpack8(w, dl);
        }
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dl[e] = 0.0f;
          if (in && d + e < d1) {
            w[e >> 1] |= (uint32_t)((const bf16_t*)p.u)[row * p.ldu + d + e] << (16 * (e & 1));
            dl[e] = load_any(p.delta, row * p.ld_delta + d + e, p.delta_f32);
          }
        }
        u[k] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      unpack8(u[k], uf);
      if (r < TT) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = dl[e] + s_bias[o * 8 + e];
          if (p.softplus) x = softplus16(x);
          sx[r][e * C8 + o] = make_float2(x, x * uf[e]);
        }
      }
      z[k] = make_uint4(0, 0, 0, 0);
      if (!LOCAL && p.z && VEC && in && d < d1) z[k] = load16_v<VEC>((const bf16_t*)p.z + row * p.ldz + fd);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int i = lane + 64 * k;
      sb[i / NS][i % NS] = p.bc_f32 ? __uint_as_float(pb[k]) : bf2f((bf16_t)pb[k]);
      if (!LOCAL) sc[i / NS][i % NS] = p.bc_f32 ? __uint_as_float(pc[k]) : bf2f((bf16_t)pc[k]);
    }
    __syncthreads();
    if (b0 + TT < c1) fetch(b0 + TT);

    // ---- walk its rows (reading the next row's values ahead of their use changed nothing, with many waves or with few).
    // Two rows a turn, but where lanes exchange their sums: the compiler leaves that loop whole.
    const int rows = b1 - b0;
#pragma unroll LOCAL || LPC == 1 ? 2 : 1
    for (int r = 0; r < rows; ++r) {
      float B[SPL], y[CPT];
#pragma unroll
      for (int s = 0; s < SPL; s += 4) *reinterpret_cast<float4*>(B + s) = *reinterpret_cast<const float4*>(&sb[r][part * SPL + s]);
      float C[SPL];
      if (!LOCAL) {
#pragma unroll
        for (int s = 0; s < SPL; s += 4) *reinterpret_cast<float4*>(C + s) = *reinterpret_cast<const float4*>(&sc[r][part * SPL + s]);
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const float2 x = sx[r][place(j)];
        if (LOCAL) sum[j] += x.x;
        float y1 = 0.0f;                           // two chains of sums
        y[j] = 0.0f;
        // (a row's decays all before the first use of one: 86 -> 96 us in pass 1)
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
          const float a = __builtin_amdgcn_exp2f(x.x * A[j][s]);
          h[j][s] = fmaf(a, h[j][s], x.y * B[s]);
          if (!LOCAL) {
            if (s & 1) y1 = fmaf(h[j][s], C[s], y1);
            else y[j] = fmaf(h[j][s], C[s], y[j]);
          }
        }
        y[j] += y1;
      }
      if (!LOCAL) {
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
#pragma unroll
          for (int o = 1; o < LPC; o <<= 1) y[j] += __shfl_xor(y[j], o, 64);
          if (part == 0) sx[r][place(j)].x = y[j];
        }
      }
    }
    __syncthreads();

    // ---- outputs of the tile
    if (!LOCAL) {
#pragma unroll
      for (int k = 0; k < E8; ++k) {
        const int piece = lane + 64 * k, r = piece / C8, c = piece % C8, d = d0 + c * 8;
        if (r >= b1 - b0 || d >= d1) continue;
        const long long row = b0 + r;
        float y[8], uf[8], zf[8];
        unpack8(u[k], uf);
        if (cut) z[k] = down16(z[k], back);
        unpack8(z[k], zf);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = sx[r][e * C8 + c].x;
          if (p.Dskip) y[e] = fmaf(s_skip[c * 8 + e], uf[e], y[e]);
          if (p.z && VEC) y[e] *= silu16(zf[e]);
        }
        if (p.z && !VEC) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (d + e < d1) y[e] *= silu16(bf2f(((const bf16_t*)p.z)[row * p.ldz + d + e]));
        }
        bf16_t* o = (bf16_t*)p.y + row * p.ldy + d;
        if (VEC == 2) {
          *reinterpret_cast<uint4*>(o) = pack8(y);
        } else if (VEC == 1 && (!cut || back == 0)) {
          store16_at(o, pack8(y));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (d + e < d1) o[e] = f2bf(y[e]);
        }
      }
      __syncthreads();
    }
  }
  if (LOCAL) {
    store_h(ck.h + (q.place + q.j + 1) * dn);
    if (part == 0) {
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        if (channel(j) < d1) ck.s[(long long)(q.place + q.j + 1) * p.D + channel(j)] = sum[j];
    }
    if (blockIdx.y == 0 && lane == 0) {
      if (q.j == 0) ck.kind[q.place] = 0;
      ck.kind[q.place + q.j + 1] = q.j > 0;
    }
  } else if (p.state && q.j + 1 == q.c) {
    store_h(state);
  }
}

// The states at the chunks' starts: a lane per channel and state walks the places of all sequences, 16 at a time, the
// next 16 under way before this ones' stores (loads that were asked for after a store wait for it). 256 places of
// 640 x 16 states: 8, 16, 32 at a time 44, 40, 37 us, this 33; 74 places of 2560 x 16 states 13.5 us. Bound: the latency
// of its loads, which few channels leave bare.
__global__ __launch_bounds__(64) void ssm_carry_kernel(const ActhSsmScanDesc p, const Chunks ck) {
  const int n = min(chunk_find(p, ck, -1).place, ck.places);
  const long long i = (long long)blockIdx.x * 64 + threadIdx.x, dn = (long long)p.D * p.N;
  if (i >= dn || n < 1) return;
  const int d = (int)(i / p.N);
  const float A = p.A[i] * kLog2e;
  constexpr int B = 16;
  float e[2][B], s[2][B], h = 0.0f;
  int kind[2][B];
  auto load = [&](int f, int k) {
#pragma unroll
    for (int v = 0; v < B; ++v) {
      const long long at = min(k + v, n - 1);
      e[f][v] = ck.h[at * dn + i];
      s[f][v] = ck.s[at * p.D + d];
      kind[f][v] = ck.kind[at];
    }
  };
  auto walk = [&](int f, int k) {
#pragma unroll
    for (int v = 0; v < B; ++v) {
      if (k + v >= n) break;
      // a chunk's decay as two factors, its root: whole, it leaves fp32 where its product with h does not, and h = 0
      // stays 0 under any growth
      const float root = __builtin_amdgcn_exp2f(0.5f * A * s[f][v]);
      const float grown = h == 0.0f ? 0.0f : root * (root * h);
      h = kind[f][v] ? e[f][v] + grown : e[f][v];
      if (kind[f][v]) ck.h[(long long)(k + v) * dn + i] = h;
    }
  };
  load(0, 0);
  for (int k = 0; k < n; k += 2 * B) {
    load(1, k + B);
    walk(0, k);
    load(0, k + 2 * B);
    walk(1, k + B);
  }
}

constexpr int STEPS = 2;                           // 512 sequences x 5120 channels x 16 states: 1, 2, 4, 8: 87, 72, 75, 93 us

// One row a sequence: a lane holds VN states of one channel (VN = 4: a 16-byte load), LPC lanes a channel, and takes SEQS
// sequences, all of whose loads are under way before the first is used, so that A is read once for them. VBC: four
// values of B (and of C) in one load. Bound: the states' bytes, in and out (512 x 5120 x 16 states: 72 us,
// 4.9 TB/s); few rows: the launch (4.2 us).
template <int VN, int LPC, int SEQS, bool VBC>
__global__ __launch_bounds__(256) void ssm_step_kernel(const ActhSsmScanDesc p) {
  const int nb = (p.D * LPC + 255) / 256;          // channel blocks, the fastest: a sequence's states one after the other
  const int bs = blockIdx.x / nb, at = (blockIdx.x - bs * nb) * 256 + threadIdx.x;
  const int d = at / LPC, part = at % LPC;
  const bool in = d < p.D;
  const int dd = in ? d : 0, n0 = part * VN, g = dd / (p.D / p.G);
  const bool on = in && n0 < p.N;                  // N % VN == 0
  const int nn = on ? n0 : 0;                      // lanes without a state of their own read the first ones
  const int r0 = bs * SEQS;

  int slot[SEQS];
  bool kept[SEQS], live[SEQS];
  float h[SEQS][VN];
  uint32_t dr[SEQS], br[SEQS][VN], cr[SEQS][VN];   // raw: a conversion here would wait for its load
  bf16_t ur[SEQS], zr[SEQS];
#pragma unroll
  for (int k = 0; k < SEQS; ++k) {
    const int r = min(r0 + k, p.T - 1);
    const Seq q = seq_of(p, r);
    live[k] = r0 + k < p.T && (!p.slots || q.slot >= 0);
    slot[k] = q.slot;
    kept[k] = seq_kept(p, q);
    const long long row = r;
    const float* st = p.state + (q.slot < 0 ? 0 : q.slot) * p.ld_slot + (long long)dd * p.N + nn;
#pragma unroll
    for (int v = 0; v < VN; ++v) h[k][v] = 0.0f;
    if (kept[k]) {
      if constexpr (VN == 4) *reinterpret_cast<float4*>(h[k]) = *reinterpret_cast<const float4*>(st);
      else h[k][0] = st[0];
    }
    ur[k] = ((const bf16_t*)p.u)[row * p.ldu + dd];
    zr[k] = 0;
    if (p.z) zr[k] = ((const bf16_t*)p.z)[row * p.ldz + dd];
    if (p.delta_f32) dr[k] = ((const uint32_t*)p.delta)[row * p.ld_delta + dd];
    else dr[k] = ((const bf16_t*)p.delta)[row * p.ld_delta + dd];
    const long long ob = row * p.ldb + g * p.N + nn, oc = row * p.ldc + g * p.N + nn;
    if constexpr (VBC) {
      if (p.bc_f32) {
        *reinterpret_cast<uint4*>(br[k]) = *reinterpret_cast<const uint4*>((const uint32_t*)p.B + ob);
        *reinterpret_cast<uint4*>(cr[k]) = *reinterpret_cast<const uint4*>((const uint32_t*)p.C + oc);
      } else {
        *reinterpret_cast<uint2*>(br[k]) = *reinterpret_cast<const uint2*>((const bf16_t*)p.B + ob);
        *reinterpret_cast<uint2*>(cr[k]) = *reinterpret_cast<const uint2*>((const bf16_t*)p.C + oc);
      }
    } else {
#pragma unroll
      for (int v = 0; v < VN; ++v) {
        if (p.bc_f32) {
          br[k][v] = ((const uint32_t*)p.B)[ob + v];
          cr[k][v] = ((const uint32_t*)p.C)[oc + v];
        } else {
          br[k][v] = ((const bf16_t*)p.B)[ob + v];
          cr[k][v] = ((const bf16_t*)p.C)[oc + v];
        }
      }
    }
  }
  float A[VN];
#pragma unroll
  for (int v = 0; v < VN; ++v) A[v] = p.A[(long long)dd * p.N + nn + v] * kLog2e;
  const float bias = p.delta_bias ? p.delta_bias[dd] : 0.0f, skip = p.Dskip ? p.Dskip[dd] : 0.0f;

#pragma unroll
  for (int k = 0; k < SEQS; ++k) {
    if (!live[k]) continue;
    float B[VN], C[VN];
#pragma unroll
    for (int v = 0; v < VN; ++v) {
      if (p.bc_f32) {
        B[v] = __uint_as_float(br[k][v]);
        C[v] = __uint_as_float(cr[k][v]);
      } else if constexpr (VBC) {
        B[v] = v & 1 ? hi16f(br[k][v >> 1]) : lo16f(br[k][v >> 1]);
        C[v] = v & 1 ? hi16f(cr[k][v >> 1]) : lo16f(cr[k][v >> 1]);
      } else {
        B[v] = bf2f((bf16_t)br[k][v]);
        C[v] = bf2f((bf16_t)cr[k][v]);
      }
    }
    float dt = (p.delta_f32 ? __uint_as_float(dr[k]) : bf2f((bf16_t)dr[k])) + bias;
    const float u = bf2f(ur[k]);
    if (p.softplus) dt = softplus16(dt);
    const float du = dt * u;
    float y = 0.0f;
#pragma unroll
    for (int v = 0; v < VN; ++v) {
      h[k][v] = fmaf(__builtin_amdgcn_exp2f(dt * A[v]), h[k][v], du * B[v]);
      y = fmaf(h[k][v], C[v], y);
    }
    if (!on) y = 0.0f;
#pragma unroll
    for (int o = 1; o < LPC; o <<= 1) y += __shfl_xor(y, o, 64);
    if (on && p.state && slot[k] >= 0) {
      float* st = p.state + slot[k] * p.ld_slot + (long long)dd * p.N + nn;
      if constexpr (VN == 4) *reinterpret_cast<float4*>(st) = make_float4(h[k][0], h[k][1], h[k][2], h[k][3]);
      else st[0] = h[k][0];
    }
    if (in && part == 0) {
      y = fmaf(skip, u, y);
      if (p.z) y *= silu16(bf2f(zr[k]));
      ((bf16_t*)p.y)[(long long)(r0 + k) * p.ldy + dd] = f2bf(y);
    }
  }
}

template <int VN, int LPC, int SEQS, bool VBC>
void launch_step2(const ActhSsmScanDesc& d, hipStream_t stream) {
  const unsigned bx = (unsigned)((d.D * LPC + 255) / 256);
  const int rows = launch_rows(bx), bsz = d.bc_f32 ? 4 : 2;
  for (int t0 = 0; t0 < d.T; t0 += rows) {
    ActhSsmScanDesc s = step_rows(d, t0, d.T - t0 < rows ? d.T - t0 : rows);
    s.u = (const bf16_t*)d.u + t0 * d.ldu;
    s.delta = (const char*)d.delta + t0 * d.ld_delta * (d.delta_f32 ? 4 : 2);
    s.B = (const char*)d.B + t0 * d.ldb * bsz;
    s.C = (const char*)d.C + t0 * d.ldc * bsz;
    if (d.z) s.z = (const bf16_t*)d.z + t0 * d.ldz;
    s.y = (bf16_t*)d.y + t0 * d.ldy;
    ssm_step_kernel<VN, LPC, SEQS, VBC><<<(unsigned)((s.T + SEQS - 1) / SEQS) * bx, 256, 0, stream>>>(s);
  }
}

// several sequences a lane once there are enough lanes (four waves a SIMD) to fill the chip without it. One against two: 512 x
// 5120 66 and 60 us, 64 x 5120 11.2 and 9.8, 40 x 2560 5.6 and 5.6, 70001 x 8 88 and 66, 20000 x 24 29 and 23 (in a graph).
template <int VN, int LPC>
void launch_step(const ActhSsmScanDesc& d, bool vbc, hipStream_t stream) {
  const bool many = (long long)d.D * LPC * (d.T / STEPS) >= 64 * 4096;
  if constexpr (VN == 4) {
    if (vbc) many ? launch_step2<VN, LPC, STEPS, true>(d, stream) : launch_step2<VN, LPC, 1, true>(d, stream);
    else many ? launch_step2<VN, LPC, STEPS, false>(d, stream) : launch_step2<VN, LPC, 1, false>(d, stream);
  } else {
    many ? launch_step2<VN, LPC, STEPS, false>(d, stream) : launch_step2<VN, LPC, 1, false>(d, stream);
  }
}

// Few rows and channels: two lanes a channel. One against two: 300 x 640 25.1 and 23.3 us, 2000 x 1280 65 and 52, 8192 x 640
// 91 and 82; 4096 x 2048 96 and 99, 16384 x 640 127 and 130, 8192 x 2560 175 and 208.
bool scan_small(int N, int T, int D) { return N > 8 && N <= 16 && (long long)T / 64 * ((D + 63) / 64) < 2048; }

// channels a wave takes
int scan_cb(int N, int T, int D) { return N <= 16 ? (scan_small(N, T, D) ? 32 : 64) : N <= 32 ? 32 : 16; }

// Chunks that give one round of the three waves that fit each of the 1024 SIMDs. Ragged ones, which differ in length, are
// made half as long (16384 x 5120 in 19 sequences: 775 -> 675 us), but not under 112 rows, where pass 1 leaves out too
// little (8192 x 2560 in 8: 173 us, of 64 rows 194). Few rows: chunks of 16, each wave being mostly latency (300 x 640 of
// 64, 32, 16 rows: 49, 31, 23 us).
constexpr int MINLEN = 16;
Chunks plan(int T, int D, int N, int G, int nseq, int ragged) {
  Chunks c{};
  const int cb = scan_cb(N, T, D);
  const long long waves = (long long)G * ((D / G + cb - 1) / cb);
  const int L = ragged ? T : T / nseq;             // the longest sequence there can be
  long long n = 3 * 1024 / waves;                  // chunks of all rows
  if (!ragged) n /= nseq;                          // of one sequence
  if (n < 1) n = 1;
  long long len = (L + n - 1) / n;
  if (ragged && len > 112) len = len / 2 > 112 ? len / 2 : 112;
  len = (len + TT - 1) / TT * TT;
  if (len < MINLEN) len = MINLEN;
  if (L <= 2 * MINLEN || len >= L) {
    c.len = L;
    c.n = nseq;
    return c;
  }
  c.len = (int)len;
  if (ragged) {
    c.n = (int)(T / len + nseq);
    c.places = (int)(2 * (T / len));               // a sequence of several chunks is longer than one
  } else {
    c.n = c.places = (int)((L + len - 1) / len * nseq);
  }
  return c;
}

template <int SPL, int LPC, int CPT, int VEC>
void launch_scan(const ActhSsmScanDesc& d, const Chunks& ck, hipStream_t stream) {
  constexpr int CB = 64 / LPC * CPT;
  const dim3 grid((unsigned)ck.n, (unsigned)(d.G * ((d.D / d.G + CB - 1) / CB)));
  if (ck.places) {
    const long long dn = (long long)d.D * d.N;
    ssm_scan_kernel<SPL, LPC, CPT, true, VEC><<<grid, 64, 0, stream>>>(d, ck);
    ssm_carry_kernel<<<(unsigned)((dn + 63) / 64), 64, 0, stream>>>(d, ck);
  }
  ssm_scan_kernel<SPL, LPC, CPT, false, VEC><<<grid, 64, 0, stream>>>(d, ck);
}

template <int VEC>
void launch_scan_n(const ActhSsmScanDesc& d, const Chunks& ck, hipStream_t stream) {
  if (d.N <= 8) launch_scan<8, 1, 1, VEC>(d, ck, stream);
  else if (scan_small(d.N, d.T, d.D)) launch_scan<8, 2, 1, VEC>(d, ck, stream);
  else if (d.N <= 16) launch_scan<16, 1, 1, VEC>(d, ck, stream);
  else if (d.N <= 32) launch_scan<16, 2, 1, VEC>(d, ck, stream);
  else launch_scan<16, 4, 1, VEC>(d, ck, stream);
}

bool al16(const void* p, long long ld_bytes) { return !p || (((uintptr_t)p | (uintptr_t)ld_bytes) % 16) == 0; }

// sequences: nseq >= 1 ranges of T rows; without starts they are equal, so nseq divides T
bool seqs_ok(int T, int nseq, const int* starts, const int* slots, const void* state, int nslots) {
  if (nseq < 1 || (!starts && T % nseq)) return false;
  if (slots && !state) return false;
  if (state && (nslots < 1 || (!slots && nslots < nseq))) return false;
  return true;
}

}  // namespace

extern "C" int acth_causal_conv(const ActhCausalConvDesc* d, hipStream_t stream) {
  if (!d || d->T < 0) return ACTH_EINVAL;
  if (d->T == 0) return ACTH_OK;
  if (d->T > (1 << 28) || d->nseq > (1 << 28) || d->D > (1 << 18)) return ACTH_EINVAL;
  if (!d->x || !d->w || !d->y || d->D < 1 || d->W < 2 || d->W > 4) return ACTH_EINVAL;
  if (!seqs_ok(d->T, d->nseq, d->starts, d->slots, d->state, d->nslots)) return ACTH_EINVAL;
  if ((d->T > 1 && (d->ldx < d->D || d->ldy < d->D)) || (d->state && d->ld_slot < (long long)(d->W - 1) * d->D))
    return ACTH_EINVAL;
  const bool vec = d->D >= 8;
  if (vec) {
    if (d->W == 2) launch_conv<8, 2>(*d, stream);
    else if (d->W == 3) launch_conv<8, 3>(*d, stream);
    else launch_conv<8, 4>(*d, stream);
  } else {
    if (d->W == 2) launch_conv<1, 2>(*d, stream);
    else if (d->W == 3) launch_conv<1, 3>(*d, stream);
    else launch_conv<1, 4>(*d, stream);
  }
  ACTH_CHECK_LAUNCH();
  return ACTH_OK;
}

extern "C" size_t acth_ssm_scan_workspace_size(int T, int D, int N, int G, int nseq, int ragged) {
  if (T < 1 || D < 1 || N < 1 || N > 64 || G < 1 || D % G || nseq < 1 || (!ragged && T % nseq)) return 0;
  const Chunks c = plan(T, D, N, G, nseq, ragged);
  return (size_t)c.places * ((size_t)D * N + D + 1) * 4;
}

extern "C" int acth_ssm_scan(const ActhSsmScanDesc* d, hipStream_t stream) {
  if (!d || d->T < 0) return ACTH_EINVAL;
  if (d->T == 0) return ACTH_OK;
  if (d->T > (1 << 28) || d->nseq > (1 << 28) || d->D > (1 << 18)) return ACTH_EINVAL;
  if (!d->u || !d->delta || !d->A || !d->B || !d->C || !d->y) return ACTH_EINVAL;
  if (d->D < 1 || d->N < 1 || d->N > 64 || d->G < 1 || d->D % d->G) return ACTH_EINVAL;
  if (!seqs_ok(d->T, d->nseq, d->starts, d->slots, d->state, d->nslots)) return ACTH_EINVAL;
  const long long gn = (long long)d->G * d->N;
  if (d->T > 1 && (d->ldu < d->D || d->ld_delta < d->D || d->ldy < d->D || (d->z && d->ldz < d->D) || d->ldb < gn ||
                   d->ldc < gn)) return ACTH_EINVAL;
  if (d->state && d->ld_slot < (long long)d->D * d->N) return ACTH_EINVAL;
  if (!d->starts && d->nseq == d->T) {
    const int bsz = d->bc_f32 ? 4 : 2;             // four values of B and of C in one load
    const bool vbc = (((uintptr_t)d->B | (uintptr_t)d->C | (uintptr_t)(d->ldb * bsz) | (uintptr_t)(d->ldc * bsz)) % (4 * bsz)) == 0;
    if (d->N % 4 == 0 && al16(d->state, d->ld_slot * 4)) {
      if (d->N <= 8) launch_step<4, 2>(*d, vbc, stream);
      else if (d->N <= 16) launch_step<4, 4>(*d, vbc, stream);
      else if (d->N <= 32) launch_step<4, 8>(*d, vbc, stream);
      else launch_step<4, 16>(*d, vbc, stream);
    } else {
      if (d->N <= 8) launch_step<1, 8>(*d, false, stream);
      else if (d->N <= 16) launch_step<1, 16>(*d, false, stream);
      else if (d->N <= 32) launch_step<1, 32>(*d, false, stream);
      else launch_step<1, 64>(*d, false, stream);
    }
    ACTH_CHECK_LAUNCH();
    return ACTH_OK;
  }
  Chunks ck = plan(d->T, d->D, d->N, d->G, d->nseq, d->starts != nullptr);
  const size_t need = acth_ssm_scan_workspace_size(d->T, d->D, d->N, d->G, d->nseq, d->starts != nullptr);
  if (need) {
    if (!d->ws || d->ws_bytes < (long long)need) return ACTH_EINVAL;
    ck.h = d->ws;
    ck.s = ck.h + (size_t)ck.places * d->D * d->N;
    ck.kind = (int*)(ck.s + (size_t)ck.places * d->D);
  }
  if (d->G * ((d->D / d->G + 15) / 16) > 65535 || ck.n >= 4 * LAUNCH) return ACTH_EINVAL;      // blocks of a launch, 64 lanes each
  const bool whole = d->D / d->G % 8 == 0 && al16(d->u, d->ldu * 2) && al16(d->delta, d->ld_delta * (d->delta_f32 ? 4 : 2)) &&
                     al16(d->z, d->ldz * 2) && al16(d->y, d->ldy * 2);
  if (whole) launch_scan_n<2>(*d, ck, stream);             // 8192 x 5120: 332 us, by the next one 352, 8192 x 5121: 362
  else if (d->D / d->G >= 8) launch_scan_n<1>(*d, ck, stream);
  else launch_scan_n<0>(*d, ck, stream);
  ACTH_CHECK_LAUNCH();
  return ACTH_OK;
}
