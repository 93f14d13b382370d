// The sequence part of a gated state-space layer, for prompts and for single tokens: the short causal convolution and
// the selective scan, over ragged sequences whose states are kept between calls.
//
//   convolution   y[t] = silu(bias + sum_j w[j] x[t - W + 1 + j])          rows before the sequence: the kept W - 1 inputs
//   scan          dt = softplus(delta + bias),  h = exp(dt A) h + dt u B,  y = (C h + D u) silu(z)
//
// Sequences are row ranges [starts[i], starts[i+1]) of one token-major tensor; `starts` lives on the device, so the
// host never learns the lengths. Everything read from it is clamped to [0, T], and a slot outside [0, nslots) marks a
// padding sequence whose rows are left alone, so no content of either can lead an access out of its tensor.
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

constexpr float kLog2e = 1.4426950408889634f;

// x / (1 + exp(-x)) with the one-step reciprocal: within 4 roundings of 2^-24, for 16-bit outputs
__device__ __forceinline__ float silu16(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// ------------------------------------------------------------------------------------------------ convolution
// VEC channels a lane (8: one 16-byte load a row; 1: any width and alignment), a wave 64 x VEC channels of 16 rows. The
// rows of a tile are loaded before the first is used; the W - 1 rows in front of it are read again (3 of 16, from L2).
// The tile that holds a sequence's first row also takes the rows that reach back into the kept inputs and writes the
// new ones, so one lane both reads and writes each kept value. Bound: HBM bandwidth.
constexpr int CT = 16;

template <int VEC>
__device__ __forceinline__ void load_c(const bf16_t* p, float* f) {
  if constexpr (VEC == 8) unpack8(*reinterpret_cast<const uint4*>(p), f);
  else f[0] = bf2f(*p);
}

template <int VEC>
__device__ __forceinline__ void store_c(bf16_t* p, const float* f) {
  if constexpr (VEC == 8) *reinterpret_cast<uint4*>(p) = pack8(f);
  else *p = f2bf(f[0]);
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
  // win: the W - 1 inputs before x, oldest first
  __device__ __forceinline__ void out(const float (*win)[VEC], const float* x, float* y) const {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float a = b[v];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) a = fmaf(w[j][v], win[j][v], a);
      a = fmaf(w[W - 1][v], x[v], a);
      y[v] = silu ? silu16(a) : a;
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

template <int VEC, int W>
__global__ __launch_bounds__(64) void causal_conv_kernel(const ActhCausalConvDesc p) {
  const int t0 = blockIdx.x * CT, t1 = min(t0 + CT, p.T);
  const int d = (blockIdx.y * 64 + threadIdx.x) * VEC;
  if (d >= p.D) return;
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
      c.out(win, xv, yv);
      store_c<VEC>(y + (long long)(t0 + k) * p.ldy, yv);
      c.shift(win, xv);
    }
    return;
  }

  int t = t0;
  while (t < t1) {
    if (q.i < 0 || q.i >= p.nseq || q.e <= t) {                  // rows that no sequence holds, or an empty sequence
      if (q.i >= p.nseq) return;
      if (q.i < 0) t = max(t, q.e);
      q = seq_of(p, q.i + 1);
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
        c.out(win, xv, yv);
        store_c<VEC>(y + (long long)r * p.ldy, yv);
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
        store_c<VEC>(st + (long long)j * p.D, nv);
      }
    }
    t = max(t, q.e);
    q = seq_of(p, q.i + 1);
    if (q.i < p.nseq && q.s > t) t = q.s;
  }
}

// one row a sequence: a lane takes VEC channels of one sequence. Bound: the kept inputs' bytes; few rows: the launch.
template <int VEC, int W>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(const ActhCausalConvDesc p) {
  const int nch = (p.D + VEC - 1) / VEC;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long r = at / nch;
  const int d = (int)(at - r * nch) * VEC;
  if (r >= p.T) return;
  const Seq q = seq_of(p, (int)r);
  if (p.slots && q.slot < 0) return;
  ConvLane<VEC, W> c;
  float win[W - 1][VEC], xv[VEC], yv[VEC];
  load_c<VEC>((const bf16_t*)p.x + r * p.ldx + d, xv);
  bf16_t* st = (bf16_t*)p.state + (long long)(q.slot < 0 ? 0 : q.slot) * p.ld_slot + d;
  const bool kept = seq_kept(p, q);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) win[j][v] = 0.0f;
    if (kept) load_c<VEC>(st + (long long)j * p.D, win[j]);
  }
  c.init(p, d);
  c.out(win, xv, yv);
  store_c<VEC>((bf16_t*)p.y + r * p.ldy + d, yv);
  if (p.state && q.slot >= 0) {
    c.shift(win, xv);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_c<VEC>(st + (long long)j * p.D, win[j]);
  }
}

template <int VEC, int W>
void launch_conv(const ActhCausalConvDesc& d, hipStream_t stream) {
  if (!d.starts && d.nseq == d.T) {
    const long long n = (long long)d.T * ((d.D + VEC - 1) / VEC);
    causal_conv_step_kernel<VEC, W><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(d);
  } else {
    const dim3 grid((unsigned)((d.T + CT - 1) / CT), (unsigned)((d.D + 64 * VEC - 1) / (64 * VEC)));
    causal_conv_kernel<VEC, W><<<grid, 64, 0, stream>>>(d);
  }
}

// ------------------------------------------------------------------------------------------------ scan

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1]. With w = 1 + e rounded and c = e - (w - 1) what the
// rounding lost, log1p(e) = log(w) + c / w + ..., and c stands for c / w: they differ by at most 2^-25 e, half a step of
// the result. So small e keep their digits, which log(1 + e) alone would lose, for 7 operations and two of the slow ones.
__device__ __forceinline__ float softplus16(float x) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
  const float w = 1.0f + e;
  const float c = e - (w - 1.0f);
  return fmaxf(x, 0.0f) + fmaf(__builtin_amdgcn_logf(w), 0.69314718055994531f, c);   // NaN passes through e
}

__device__ __forceinline__ float load_any(const void* p, long long i, int f32) {
  return f32 ? ((const float*)p)[i] : bf2f(((const bf16_t*)p)[i]);
}

// A long axis with few rows is cut into chunks of rows:
//   pass 1 (LOCAL)   every chunk from a zero state (or from the sequence that starts in it): its end state and the sum
//                    of its time steps, which gives the chunk's decay exp(A sum dt) for all states at once;
//   carry            the states at the chunks' starts, one after the other, a lane per channel and state;
//   pass 2 (FINAL)   every chunk from its true start state: outputs and kept states.
// Chunks are ranges of the row axis and not of a sequence, so their number needs no lengths; a sequence that starts
// inside a chunk replaces the state there. A chunk that ends where a sequence ends skips pass 1.
struct Chunks {
  int len, n;                                      // rows a chunk, chunks
  float* h;                                        // (n, D, N): end states, then start states, then kept states
  float* s;                                        // (n, D): sums of the time steps
};

constexpr int TT = 8;                             // rows of a tile in LDS

// A wave takes CB channels of a chunk: SPL states a lane, LPC lanes a channel, CPT channels a lane. A tile's time steps
// (softplus done once, by the staging lane) and inputs dt u sit in LDS as pairs beside the rows of B and C; the output
// takes the place of the pair that its own lane has just read. The next tile's rows are loaded while this one is
// walked. One wave a block, so no barrier waits for another wave.
// Channel c of a row lies at place (c % 8)(CB / 8) + c / 8, and rows are CB bytes further apart than they are long:
// the staging lanes, which hold 8 neighbouring channels each, then write neighbouring places (laid out by channel they
// met in 4 banks, 16 at a time), and the walking lanes read one place each.
// Bound: the vector units, a row, channel and state taking one exponential (8 clocks a wave) and four operations (4 each).
template <int SPL, int LPC, int CPT, bool LOCAL, bool VEC>
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
  __shared__ int s_ok[TT];

  const int lane = threadIdx.x;
  const int chunk = blockIdx.x;
  const int c0 = chunk * ck.len, c1 = min(c0 + ck.len, p.T);
  const int dg = p.D / p.G, nb = (dg + CB - 1) / CB;
  const int g = blockIdx.y / nb;
  const int d0 = g * dg + (blockIdx.y - g * nb) * CB, d1 = min(d0 + CB, (g + 1) * dg);

  Seq q = seq_find(p, c0);
  if (LOCAL) {
    if (c1 >= p.T) return;
    const Seq last = seq_find(p, c1);              // is the chunk's end state anybody's start state?
    if (last.i < 0 || last.i >= p.nseq || last.s >= c1 || last.e <= c1) return;
  }

  // ---- loads of a tile, held until the tile before it is done. A lane's places move down TT rows a tile. Rows behind
  // the chunk are not loaded and channels behind the wave's last read that one again: what they leave is never walked
  // or never stored. States behind the last one keep zeros.
  uint4 pu[E8], pd[E8][2];
  uint32_t pb[NB], pc[NB];                         // raw: a conversion here would wait for its load
  const int dsz = p.delta_f32 ? 4 : 2, bsz = p.bc_f32 ? 4 : 2;
  const int fr = lane / C8, fd = min(d0 + lane % C8 * 8, d1 - 8);      // (fd: with VEC, d1 - d0 is a multiple of 8)
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
          pu[k] = *reinterpret_cast<const uint4*>(at_u + (long long)(64 / C8 * k) * p.ldu);
          const uint4* f = reinterpret_cast<const uint4*>(at_d + (long long)(64 / C8 * k) * p.ld_delta * dsz);
          pd[k][0] = f[0];
          if (p.delta_f32) pd[k][1] = f[1];
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
  if (!LOCAL && q.i >= 0 && q.i < p.nseq && q.s < c0 && q.e > c0) load_h(ck.h + chunk * dn);
  pin();

  int t = c0;
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
        if (p.delta_f32) {
          dl[0] = __uint_as_float(pd[k][0].x); dl[1] = __uint_as_float(pd[k][0].y);
          dl[2] = __uint_as_float(pd[k][0].z); dl[3] = __uint_as_float(pd[k][0].w);
          dl[4] = __uint_as_float(pd[k][1].x); dl[5] = __uint_as_float(pd[k][1].y);
          dl[6] = __uint_as_float(pd[k][1].z); dl[7] = __uint_as_float(pd[k][1].w);
        } else {
          unpack8(pd[k][0], dl);
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
      if (!LOCAL && p.z && VEC && in && d < d1) z[k] = *reinterpret_cast<const uint4*>((const bf16_t*)p.z + row * p.ldz + d);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int i = lane + 64 * k;
      sb[i / NS][i % NS] = p.bc_f32 ? __uint_as_float(pb[k]) : bf2f((bf16_t)pb[k]);
      if (!LOCAL) sc[i / NS][i % NS] = p.bc_f32 ? __uint_as_float(pc[k]) : bf2f((bf16_t)pc[k]);
    }
    if (!LOCAL && lane < TT) s_ok[lane] = 0;
    __syncthreads();
    if (b0 + TT < c1) fetch(b0 + TT);

    // ---- walk its rows, sequence by sequence
    while (t < b1) {
      if (q.i >= p.nseq) { t = b1; break; }
      if (q.i < 0 || q.e <= t) {                   // rows that no sequence holds, or an empty sequence
        if (q.i < 0) t = max(t, min(q.e, b1));
        if (q.i < 0 && q.e > t) break;
        q = seq_of(p, q.i + 1);
        continue;
      }
      if (q.s > t) { t = min(q.s, b1); continue; }
      if (t == q.s) {
#pragma unroll
        for (int j = 0; j < CPT; ++j)
#pragma unroll
          for (int s = 0; s < SPL; ++s) h[j][s] = 0.0f;
        if (seq_kept(p, q)) {
          load_h(p.state + q.slot * p.ld_slot);
          pin();
        }
      }
      const int e = min(q.e, b1);
      if (!LOCAL && lane >= t - b0 && lane < e - b0) s_ok[lane] = !p.slots || q.slot >= 0;
#pragma unroll 2
      for (; t < e; ++t) {
        const int r = t - b0;
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
          float y1 = 0.0f;
          y[j] = 0.0f;
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
      if (t == q.e) {
        if (!LOCAL && p.state && q.slot >= 0) {
          // a sequence that began in another chunk: that chunk may not have read the kept state yet, so the new one
          // waits in this chunk's own workspace row (its start state has been read) for the last kernel
          store_h(q.s < c0 ? ck.h + chunk * dn : p.state + q.slot * p.ld_slot);
        }
        q = seq_of(p, q.i + 1);
      }
    }
    __syncthreads();

    // ---- outputs of the tile
    if (!LOCAL) {
#pragma unroll
      for (int k = 0; k < E8; ++k) {
        const int piece = lane + 64 * k, r = piece / C8, c = piece % C8, d = d0 + c * 8;
        if (r >= TT || !s_ok[r < TT ? r : 0] || d >= d1) continue;
        const long long row = b0 + r;
        float y[8], uf[8], zf[8];
        unpack8(u[k], uf);
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
        if constexpr (VEC) {
          *reinterpret_cast<uint4*>(o) = pack8(y);
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
    store_h(ck.h + chunk * dn);
    if (part == 0) {
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        if (channel(j) < d1) ck.s[(long long)chunk * p.D + channel(j)] = sum[j];
    }
  }
}

// The states at the chunks' starts: a lane per channel and state walks the chunks. Where a sequence starts inside a
// chunk nothing passes through it; where a chunk's end state is nobody's start state (pass 1 left it out) zero does.
__global__ __launch_bounds__(256) void ssm_carry_kernel(const ActhSsmScanDesc p, const Chunks ck) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x, dn = (long long)p.D * p.N;
  __shared__ int s_kind[256];                       // of 256 chunks: 0 end unused, 1 starts anew inside, 2 passes through
  const long long ii = i < dn ? i : 0;
  const int d = (int)(ii / p.N);
  const float A = p.A[ii] * kLog2e;
  float h = 0.0f;
  for (int b = 0; b + 1 < ck.n; b += 256) {
    __syncthreads();
    const int c = b + threadIdx.x;
    if (c + 1 < ck.n) {
      const int c0 = c * ck.len, c1 = c0 + ck.len;
      const Seq q = seq_find(p, c1);
      s_kind[threadIdx.x] = q.i < 0 || q.i >= p.nseq || q.s >= c1 || q.e <= c1 ? 0 : q.s >= c0 ? 1 : 2;
    }
    __syncthreads();
    const int n = min(256, ck.n - 1 - b);
    // loads of 8 chunks at a time, whatever their kind, so that they are all under way together
    for (int k = 0; k < n; k += 8) {
      float e[8], s[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const long long at = b + min(k + v, n - 1);
        e[v] = ck.h[at * dn + ii];
        s[v] = ck.s[at * p.D + d];
      }
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        if (k + v >= n) break;
        const int kind = s_kind[k + v];
        if (i < dn) ck.h[(b + k + v) * dn + ii] = h;
        const float keep = kind == 2 ? __builtin_amdgcn_exp2f(A * s[v]) * h : 0.0f;
        h = kind ? keep + e[v] : 0.0f;
      }
    }
  }
  if (i < dn) ck.h[(long long)(ck.n - 1) * dn + ii] = h;
}

// the kept states of the sequences that span chunks, from the workspace row of the chunk they end in
__global__ __launch_bounds__(256) void ssm_keep_kernel(const ActhSsmScanDesc p, const Chunks ck) {
  const int c = blockIdx.y, c0 = c * ck.len, c1 = min(c0 + ck.len, p.T);
  const Seq q = seq_find(p, c0);
  if (q.i < 0 || q.i >= p.nseq || q.s >= c0 || q.e <= c0 || q.e > c1 || q.slot < 0) return;
  const long long dn = (long long)p.D * p.N;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const long long i = ((long long)blockIdx.x * 16 + k) * 256 + threadIdx.x;
    if (i < dn) p.state[q.slot * p.ld_slot + i] = ck.h[c * dn + i];
  }
}

// One row a sequence: a lane holds VN states of one channel (VN = 4: a 16-byte load), LPC lanes a channel, and takes
// SEQS sequences so that A is read once for them. Bound: the states' bytes, in and out; few rows: the launch.
template <int VN, int LPC>
__global__ __launch_bounds__(256) void ssm_step_kernel(const ActhSsmScanDesc p, int seqs) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int d = (int)(at / LPC), part = (int)(at % LPC);
  const bool in = d < p.D;
  const int dd = in ? d : 0, n0 = part * VN, g = dd / (p.D / p.G);
  const bool on = in && n0 < p.N;                  // N % VN == 0
  float A[VN];
#pragma unroll
  for (int v = 0; v < VN; ++v) A[v] = on ? p.A[(long long)dd * p.N + n0 + v] * kLog2e : 0.0f;
  const float bias = p.delta_bias ? p.delta_bias[dd] : 0.0f, skip = p.Dskip ? p.Dskip[dd] : 0.0f;
  const int r1 = (int)min((long long)p.T, ((long long)blockIdx.y + 1) * seqs);
  for (int r = blockIdx.y * seqs; r < r1; ++r) {
    const Seq q = seq_of(p, r);
    if (p.slots && q.slot < 0) continue;
    const long long row = r;
    float dt = load_any(p.delta, row * p.ld_delta + dd, p.delta_f32) + bias;
    const float u = bf2f(((const bf16_t*)p.u)[row * p.ldu + dd]);
    float h[VN], B[VN], C[VN];
#pragma unroll
    for (int v = 0; v < VN; ++v) { h[v] = 0.0f; B[v] = 0.0f; C[v] = 0.0f; }
    float* st = p.state + (q.slot < 0 ? 0 : q.slot) * p.ld_slot + (long long)dd * p.N + n0;
    if (on) {
      if (seq_kept(p, q)) {
        if constexpr (VN == 4) *reinterpret_cast<float4*>(h) = *reinterpret_cast<const float4*>(st);
        else h[0] = st[0];
      }
#pragma unroll
      for (int v = 0; v < VN; ++v) {
        B[v] = load_any(p.B, row * p.ldb + g * p.N + n0 + v, p.bc_f32);
        C[v] = load_any(p.C, row * p.ldc + g * p.N + n0 + v, p.bc_f32);
      }
    }
    if (p.softplus) dt = softplus16(dt);
    const float du = dt * u;
    float y = 0.0f;
#pragma unroll
    for (int v = 0; v < VN; ++v) {
      h[v] = fmaf(__builtin_amdgcn_exp2f(dt * A[v]), h[v], du * B[v]);
      y = fmaf(h[v], C[v], y);
    }
#pragma unroll
    for (int o = 1; o < LPC; o <<= 1) y += __shfl_xor(y, o, 64);
    if (on && p.state && q.slot >= 0) {
      if constexpr (VN == 4) *reinterpret_cast<float4*>(st) = make_float4(h[0], h[1], h[2], h[3]);
      else st[0] = h[0];
    }
    if (in && part == 0) {
      y = fmaf(skip, u, y);
      if (p.z) y *= silu16(bf2f(((const bf16_t*)p.z)[row * p.ldz + dd]));
      ((bf16_t*)p.y)[row * p.ldy + dd] = f2bf(y);
    }
  }
}

template <int VN, int LPC>
void launch_step(const ActhSsmScanDesc& d, hipStream_t stream) {
  const int seqs = d.T >= 256 ? 4 : 1;
  const dim3 grid((unsigned)(((long long)d.D * LPC + 255) / 256), (unsigned)((d.T + seqs - 1) / seqs));
  ssm_step_kernel<VN, LPC><<<grid, 256, 0, stream>>>(d, seqs);
}

// channels a wave takes, by the number of states
int scan_cb(int N) { return N <= 16 ? 64 : N <= 32 ? 32 : 16; }

Chunks plan(int T, int D, int N, int G, int nseq, int ragged) {
  Chunks c{};
  const int cb = scan_cb(N);
  const long long waves = (long long)G * ((D / G + cb - 1) / cb);
  const int L = T / nseq;
  if (!ragged && (nseq == 1 ? T <= 128 : waves * nseq >= 1024 || L <= 64)) {
    c.len = L;
    c.n = nseq;
    return c;
  }
  long long n = 3072 / waves;                      // one round of the three waves that fit each of 1024 SIMDs
  if (n < 1) n = 1;
  long long len = (T + n - 1) / n;
  len = (len + 15) / 16 * 16;
  if (len < 64) len = 64;
  while (T / len >= 65535) len *= 2;               // the chunks are one launch's second dimension
  c.len = (int)len;
  c.n = (int)((T + len - 1) / len);
  return c;
}

template <int SPL, int LPC, int CPT, bool VEC>
void launch_scan(const ActhSsmScanDesc& d, const Chunks& ck, bool chunked, hipStream_t stream) {
  constexpr int CB = 64 / LPC * CPT;
  const dim3 grid((unsigned)ck.n, (unsigned)(d.G * ((d.D / d.G + CB - 1) / CB)));
  if (chunked) {
    const long long dn = (long long)d.D * d.N;
    ssm_scan_kernel<SPL, LPC, CPT, true, VEC><<<grid, 64, 0, stream>>>(d, ck);
    ssm_carry_kernel<<<(unsigned)((dn + 255) / 256), 256, 0, stream>>>(d, ck);
    ssm_scan_kernel<SPL, LPC, CPT, false, VEC><<<grid, 64, 0, stream>>>(d, ck);
    if (d.state) ssm_keep_kernel<<<dim3((unsigned)((dn + 4095) / 4096), (unsigned)ck.n), 256, 0, stream>>>(d, ck);
  } else {
    ssm_scan_kernel<SPL, LPC, CPT, false, VEC><<<grid, 64, 0, stream>>>(d, ck);
  }
}

template <bool VEC>
void launch_scan_n(const ActhSsmScanDesc& d, const Chunks& ck, bool chunked, hipStream_t stream) {
  if (d.N <= 8) launch_scan<8, 1, 1, VEC>(d, ck, chunked, stream);
  else if (d.N <= 16) launch_scan<16, 1, 1, VEC>(d, ck, chunked, stream);
  else if (d.N <= 32) launch_scan<16, 2, 1, VEC>(d, ck, chunked, stream);
  else launch_scan<16, 4, 1, VEC>(d, ck, chunked, stream);
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
  if (!d->x || !d->w || !d->y || d->D < 1 || d->W < 2 || d->W > 4) return ACTH_EINVAL;
  if (!seqs_ok(d->T, d->nseq, d->starts, d->slots, d->state, d->nslots)) return ACTH_EINVAL;
  if ((d->T > 1 && (d->ldx < d->D || d->ldy < d->D)) || (d->state && d->ld_slot < (long long)(d->W - 1) * d->D))
    return ACTH_EINVAL;
  if (d->D > (1 << 25) || (d->T + CT - 1) / CT > (1 << 30)) return ACTH_EINVAL;
  const bool vec = d->D % 8 == 0 && al16(d->x, d->ldx * 2) && al16(d->y, d->ldy * 2) && al16(d->state, d->ld_slot * 2);
  if (!vec && d->D > 65535 * 64) return ACTH_EINVAL;
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
  if (c.n < 2 || (!ragged && c.n == nseq && c.len == T / nseq)) return 0;
  return (size_t)c.n * ((size_t)D * N + D) * 4;
}

extern "C" int acth_ssm_scan(const ActhSsmScanDesc* d, hipStream_t stream) {
  if (!d || d->T < 0) return ACTH_EINVAL;
  if (d->T == 0) return ACTH_OK;
  if (!d->u || !d->delta || !d->A || !d->B || !d->C || !d->y) return ACTH_EINVAL;
  if (d->D < 1 || d->N < 1 || d->N > 64 || d->G < 1 || d->D % d->G) return ACTH_EINVAL;
  if (!seqs_ok(d->T, d->nseq, d->starts, d->slots, d->state, d->nslots)) return ACTH_EINVAL;
  const long long gn = (long long)d->G * d->N;
  if (d->T > 1 && (d->ldu < d->D || d->ld_delta < d->D || d->ldy < d->D || (d->z && d->ldz < d->D) || d->ldb < gn ||
                   d->ldc < gn)) return ACTH_EINVAL;
  if (d->state && d->ld_slot < (long long)d->D * d->N) return ACTH_EINVAL;
  if (!d->starts && d->nseq == d->T) {
    if (d->T > 65535 * 4) return ACTH_EINVAL;
    if (d->N % 4 == 0 && al16(d->state, d->ld_slot * 4)) {
      if (d->N <= 8) launch_step<4, 2>(*d, stream);
      else if (d->N <= 16) launch_step<4, 4>(*d, stream);
      else if (d->N <= 32) launch_step<4, 8>(*d, stream);
      else launch_step<4, 16>(*d, stream);
    } else {
      if (d->N <= 8) launch_step<1, 8>(*d, stream);
      else if (d->N <= 16) launch_step<1, 16>(*d, stream);
      else if (d->N <= 32) launch_step<1, 32>(*d, stream);
      else launch_step<1, 64>(*d, stream);
    }
    ACTH_CHECK_LAUNCH();
    return ACTH_OK;
  }
  Chunks ck = plan(d->T, d->D, d->N, d->G, d->nseq, d->starts != nullptr);
  const size_t need = acth_ssm_scan_workspace_size(d->T, d->D, d->N, d->G, d->nseq, d->starts != nullptr);
  if (need) {
    if (!d->ws || d->ws_bytes < (long long)need) return ACTH_EINVAL;
    ck.h = d->ws;
    ck.s = d->ws + (size_t)ck.n * d->D * d->N;
  }
  if (d->G * ((d->D / d->G + 15) / 16) > 65535) return ACTH_EINVAL;
  const bool vec = d->D / d->G % 8 == 0 && al16(d->u, d->ldu * 2) && al16(d->delta, d->ld_delta * (d->delta_f32 ? 4 : 2)) &&
                  al16(d->z, d->ldz * 2) && al16(d->y, d->ldy * 2);
  if (vec) launch_scan_n<true>(*d, ck, need != 0, stream);
  else launch_scan_n<false>(*d, ck, need != 0, stream);
  ACTH_CHECK_LAUNCH();
  return ACTH_OK;
}
