// Linear attention with a decay per head.  Per batch row and head, over tokens t:
//
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T        (state dk x dv, fp32)
//   o_t = scale * q_t S_t
//
// in chunks of C tokens.  With G the inclusive sum of g inside the chunk, T its last value and H
// the state before the chunk,
//
//   o_i = scale * ( e^{G_i} q_i H + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j )
//   H  <- e^T H + sum_j e^{T - G_j} k_j v_j^T
//
// Every exponent is <= 0 for g <= 0.  The gradients are three more runs of the same recurrence, two
// of them from the last token to the first ("reverse": pairs j >= i, output weight e^{T - G_i},
// update weight e^{G_j}):
//
//   dq = run(q: do, k: v, v: k)   dv = reverse run(q: k, k: q, v: do)   dk = reverse run(q: v, k: do, v: q)
//
// The state of the dv run, times scale, is the gradient of the state (dS_0 at its end); and with
// D_i = q_i . dq_i - k_i . dk_i, dg_t = sum_{i >= t} D_i + <dS_last, S_last>: each weight e^{G_i - G_j}
// holds g_t once for every pair j < t <= i, and the sums telescope to the pairs that span t.
#pragma once
#include <type_traits>

#include "ss_common.cuh"

namespace ssb {

// one run of the recurrence over a (batch, seqlen, heads) problem
struct LinPass {
  const void *q, *k, *v;
  void* o;
  int64_t qb, ql, qh, kb, kl, kh, vb, vl, vh, ob, ol, oh;  // element strides of batch, token, head
  int rq, rk, rv;      // heads that share one head of q, k, v
  int dk, dv;
  int reverse;
  int o_f32;           // o is fp32 (per-head parts of a gradient that a later kernel sums), else the I/O dtype
  float scale;
  const float* s_in;   // initial state, nullable: element (i, j) at i * s_row + j * s_col of a (dk * dv) block per (b, h)
  float s_in_scale;
  float* s_out;        // final state, nullable
  float s_out_scale;
  int s_row, s_col;
  // dot[tile][b][h][t] = sum over the tile's output columns of p[.., t, ..] * o (before rounding); for fp32 I/O
  // these are doubles (LinDot), since the decays' gradient is what is left of them when they cancel
  const void* p;
  int64_t pb, pl, ph;
  int rp;
  float* dot;
  float* sum;          // segments' own states, then the states before them: [b * h][segment][dk * dv]; null for one segment
};

template <typename IT> using LinDot = typename std::conditional<sizeof(IT) == 4, double, float>::type;

constexpr int kLinMaxPasses = 3;

struct LinK {
  LinPass pass[kLinMaxPasses];
  const void* g;       // log decay: I/O dtype or fp32
  int g_f32;
  int64_t gb, gl, gh;
  const int* lens;     // nullable
  float* seg_decay;    // [direction][b * h][segment]: the segment's total log decay
  int batch, seqlen, heads;
  int segs, seg_first, seg_chunks;  // segments of the sequence, chunks of the first and of each other
};

// log decays below this act as a reset: e^x is 0 in fp32 already, and sums of -1e4 stay exact
constexpr float kLinReset = -1.0e4f;
constexpr float kLinZeroBelow = -104.f;  // e^x rounds to zero in fp32

__device__ __forceinline__ float lin_decay(const LinK& P, int b, int t, int h, bool bf16) {
  const int64_t at = (int64_t)b * P.gb + (int64_t)t * P.gl + (int64_t)h * P.gh;
  float g;
  if (P.g_f32) g = static_cast<const float*>(P.g)[at];
  else if (bf16) g = to_f<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(P.g)[at]);
  else g = to_f<__half>(static_cast<const __half*>(P.g)[at]);
  return g < kLinReset ? kLinReset : g;  // keeps NaN
}

// ------------------------------------------------------------------ fp32 units, any size and stride
// One CTA per (segment, batch row and head, 64 value columns, pass); chunks of 64 tokens in shared
// memory as fp32, each thread of a group of 128 an 8 x 4 tile of a product (4 x 4 tiles wait for shared memory
// twice as long).  One group makes the scores while the other multiplies with the state, both take half of
// the tokens in P V, then one updates the state while the other writes the outputs.  This path serves fp32 I/O, where
// 16-bit tensor-core operands would lose half the mantissa.  A chunk is a chain of short steps with
// barriers between them, so heads of at most DMAX = 64 run two CTAs on an SM (and are cut into twice the
// segments); wider ones fill its shared memory alone.  8 x 1024 tokens of 12 heads of 64 x 64 take 150 us forward
// (21 TFLOP/s) and 326 us backward, 296 and 683 us with one CTA of 4 x 4 tiles to an SM.  What bounds a chunk now
// is no single unit: of the main pass's cycles 64 % issue an instruction and 58 % move a wavefront of shared memory
// (12 of them for 32 multiply-adds of a warp), and 16 warps an SM wait for one another at the barriers.
constexpr int kLsC = 64;          // tokens of a chunk
constexpr int kLsN = 64;          // value columns of a CTA
constexpr int kLsThreads = 256;
constexpr int kLsLd = 68;         // row stride (floats): 16-byte aligned, rows 4 banks apart
constexpr int kLinMaxDim = 128;

template <int DMAX>
struct LsSmem {
  float qt[DMAX][kLsLd];        // [d][token]
  float kt[DMAX][kLsLd];
  float v[kLsC][kLsLd];         // [token][column]
  float h[DMAX][kLsLd];         // [d][column]
  float at[kLsC][kLsLd];        // weighted scores, [j][i]
  float gh[kLsC], gl[kLsC];     // G log2 e in two parts
  float w_out[kLsC], w_upd[kLsC];
  double total;
};

template <typename IT, int DMAX, bool STATE_ONLY>
__global__ void __launch_bounds__(kLsThreads, 128 / DMAX) linear_simt_kernel(const __grid_constant__ LinK P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  LsSmem<DMAX>& S = *reinterpret_cast<LsSmem<DMAX>*>(smem_raw);
  constexpr int tiles = DMAX / kLsN;
  const LinPass& A = P.pass[blockIdx.y / tiles];
  const int tile = blockIdx.y % tiles;
  const int n0 = tile * kLsN;
  const int dk = A.dk, dv = A.dv;
  if (n0 >= dv) return;
  const int nv = min(kLsN, dv - n0);
  const int bh = blockIdx.x % (P.batch * P.heads), seg = blockIdx.x / (P.batch * P.heads);
  if (STATE_ONLY) griddep_launch_dependents();
  else if (seg > 0) griddep_wait();  // the first segment needs nothing of the passes before
  if (STATE_ONLY && seg == P.segs - 1) return;  // nothing follows the last segment
  const int b = bh / P.heads, head = bh % P.heads;
  const int len = P.lens ? max(0, min(P.lens[b], P.seqlen)) : P.seqlen;
  const int n_chunks = (P.seqlen + kLsC - 1) / kLsC, n_live = (len + kLsC - 1) / kLsC;
  const int c0 = seg ? P.seg_first + (seg - 1) * P.seg_chunks : 0,
            c1 = min(seg ? c0 + P.seg_chunks : P.seg_first, n_chunks);
  const IT* q = static_cast<const IT*>(A.q) + (int64_t)b * A.qb + (int64_t)(head / A.rq) * A.qh;
  const IT* k = static_cast<const IT*>(A.k) + (int64_t)b * A.kb + (int64_t)(head / A.rk) * A.kh;
  const IT* v = static_cast<const IT*>(A.v) + (int64_t)b * A.vb + (int64_t)(head / A.rv) * A.vh + n0;
  const int tid = threadIdx.x;
  const bool second = tid >= kLsThreads / 2;       // the group that makes the outputs
  const int ti = (tid / 16 & 7) * 8, tj = tid % 16 * 4;  // 8 x 4 tile of a group's 64 x 64 product
  const int64_t block = (int64_t)dk * dv;
  // outputs as vectors of 4 fp32 values
  const bool o_vec = (A.o_f32 || sizeof(IT) == 4) && dv % 4 == 0 && (reinterpret_cast<uintptr_t>(A.o) & 15) == 0 &&
                     ((A.ob | A.ol | A.oh) & 3) == 0;

  // the state before this segment: the initial state, or what it and the earlier segments fold to
  for (int e = tid; e < DMAX * kLsN; e += kLsThreads) {
    const int i = e / kLsN, j = e % kLsN;
    float s = 0.f;
    if (!STATE_ONLY && i < dk && j < nv) {
      if (seg > 0) s = A.sum[((int64_t)bh * P.segs + seg) * block + (int64_t)i * dv + n0 + j];
      else if (A.s_in) s = A.s_in_scale * A.s_in[bh * block + (int64_t)i * A.s_row + (int64_t)(n0 + j) * A.s_col];
    }
    S.h[i][j] = s;
  }
  double seg_total = 0.0;

  // A chunk's inputs in registers, 16 threads a token and 4 tokens a thread: all of them under way at once, and
  // the next chunk's while this one is computed
  float xq[4][STATE_ONLY ? 1 : DMAX / 16], xk[4][DMAX / 16], xv[4][kLsN / 16], xg[2];
  auto first_token = [&](int c) { return (A.reverse ? n_live - 1 - c : c) * kLsC; };
  auto load = [&](int c) {
    const int t0 = first_token(c), m = c < min(c1, n_live) ? min(kLsC, len - t0) : 0;
    auto fetch = [&](auto& x, const IT* p, int64_t stride, int n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = tid / 16 + 16 * i;
#pragma unroll
        for (int j = 0; j < (int)(sizeof(x[0]) / sizeof(float)); ++j) {
          const int d = tid % 16 + 16 * j;
          x[i][j] = t < m && d < n ? to_f<IT>(p[(int64_t)(t0 + t) * stride + d]) : 0.f;
        }
      }
    };
    if constexpr (!STATE_ONLY) fetch(xq, q, A.ql, dk);
    fetch(xk, k, A.kl, dk);
    fetch(xv, v, A.vl, nv);
    constexpr bool bf = std::is_same<IT, __nv_bfloat16>::value;
    if (tid < 32)
#pragma unroll
      for (int r = 0; r < 2; ++r) xg[r] = 2 * tid + r < m ? lin_decay(P, b, t0 + 2 * tid + r, head, bf) : 0.f;
  };
  constexpr bool kAhead = DMAX > 64;  // beside a second CTA the registers are worth more
  if (kAhead) load(c0);

  for (int c = c0; c < (STATE_ONLY ? min(c1, n_live) : c1); ++c) {
    if (!STATE_ONLY && c >= n_live) {  // behind the row's end: zero outputs
      for (int e = tid; e < kLsC * kLsN; e += kLsThreads) {
        const int t = c * kLsC + e / kLsN, j = e % kLsN;
        if (t < P.seqlen && j < nv) {
          const int64_t at = (int64_t)b * A.ob + (int64_t)t * A.ol + (int64_t)head * A.oh + n0 + j;
          if (A.o_f32) static_cast<float*>(A.o)[at] = 0.f;
          else static_cast<IT*>(A.o)[at] = zero_v<IT>();
        }
      }
      if (A.dot && tid < kLsC && c * kLsC + tid < P.seqlen)
        reinterpret_cast<LinDot<IT>*>(A.dot)[(((int64_t)tile * P.batch + b) * P.heads + head) * P.seqlen + c * kLsC + tid] = 0;
      continue;
    }
    const int t0 = first_token(c);
    const int m = min(kLsC, len - t0);  // valid tokens
    if (!kAhead) load(c);
    __syncthreads();                    // the chunk before is done with shared memory
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = tid / 16 + 16 * i, d = tid % 16;
#pragma unroll
      for (int j = 0; j < DMAX / 16; ++j) {
        if constexpr (!STATE_ONLY) S.qt[d + 16 * j][t] = xq[i][j];
        S.kt[d + 16 * j][t] = xk[i][j];
      }
#pragma unroll
      for (int j = 0; j < kLsN / 16; ++j) S.v[t][d + 16 * j] = xv[i][j];
    }
    if (tid < 32) {  // inclusive sums of two tokens a lane, in 64 bits: differences stay exact behind a reset
      const double g0 = xg[0], g1 = xg[1];
      double s = g0 + g1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, s, o);
        if (tid >= o) s += x;
      }
      const double T = __shfl_sync(0xffffffffu, s, 31);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const double G = r ? s : s - g1;
        const int t = 2 * tid + r;
        const double g2 = G * 1.4426950408889634;
        S.gh[t] = (float)g2;
        S.gl[t] = (float)(g2 - (double)(float)g2);
        const float a = expf((float)G), z = expf((float)(T - G));
        S.w_out[t] = A.reverse ? z : a;
        S.w_upd[t] = t < m ? (A.reverse ? a : z) : 0.f;
      }
      if (tid == 0) S.total = T;
    }
    __syncthreads();
    if (kAhead) load(c + 1);
    seg_total += S.total;
    if constexpr (!STATE_ONLY) {
      // acc += a[n][ti ..] b[n][tj ..] over n in [n0, n1), both multiples of 8
      float acc[8][4] = {};
      auto product = [&](const float (*a)[kLsLd], const float (*b)[kLsLd], int n0, int n1) {
        for (int n = n0; n < n1; n += 4) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(&a[n + r][ti]), z = *reinterpret_cast<const float4*>(&a[n + r][ti + 4]);
            const float4 y = *reinterpret_cast<const float4*>(&b[n + r][tj]);
            const float xa[8] = {x.x, x.y, x.z, x.w, z.x, z.y, z.z, z.w}, ya[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xa[i], ya[j], acc[i][j]);
          }
        }
      };
      const int dk8 = (dk + 7) & ~7;  // rows behind dk are zero
      if (second) {  // e^{G_i} q_i H
        product(S.qt, S.h, 0, dk8);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] *= S.w_out[ti + i];
      } else {  // scores, weighted by the decay between the two tokens
        product(S.qt, S.kt, 0, dk8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = tj + j;
          const float gh = S.gh[n], gl = S.gl[n];
          float w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = ti + i;
            const bool on = A.reverse ? n >= r : n <= r;
            const float d = (S.gh[r] - gh) + (S.gl[r] - gl);  // the difference of the sums, rounded once
            w[i] = on && n < m ? acc[i][j] * ex2(A.reverse ? -d : d) : 0.f;
          }
          *reinterpret_cast<float4*>(&S.at[n][ti]) = make_float4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<float4*>(&S.at[n][ti + 4]) = make_float4(w[4], w[5], w[6], w[7]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
      }
      __syncthreads();  // scores written, H and q read
      // each group's half of the tokens; a warp's 16 rows need none on the far side of the diagonal
      const int r16 = ti & ~15, half = second ? kLsC / 2 : 0;
      product(S.at, S.v, A.reverse ? max(half, r16) : half, A.reverse ? half + kLsC / 2 : min(half + kLsC / 2, r16 + 16));
      float(*part)[kLsLd] = S.qt;
      if (!second) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4*>(&part[ti + i][tj]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
      }
      __syncthreads();
      if (second) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = t0 + ti + i;
          const bool on = ti + i < m;
          LinDot<IT> dot = 0;
          if (t < P.seqlen) {
            const float4 x = *reinterpret_cast<const float4*>(&part[ti + i][tj]);
            const float xa[4] = {x.x, x.y, x.z, x.w};
            const int64_t at = (int64_t)b * A.ob + (int64_t)t * A.ol + (int64_t)head * A.oh + n0 + tj;
            float r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = on ? A.scale * (acc[i][j] + xa[j]) : 0.f;
            if (o_vec) {
              if (tj < nv) *reinterpret_cast<float4*>(static_cast<float*>(A.o) + at) = make_float4(r[0], r[1], r[2], r[3]);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (tj + j < nv) {
                  if (A.o_f32) static_cast<float*>(A.o)[at + j] = r[j];
                  else static_cast<IT*>(A.o)[at + j] = from_f<IT>(r[j]);
                }
            }
            if (A.dot && on) {
              const IT* p = static_cast<const IT*>(A.p) + (int64_t)b * A.pb + (int64_t)t * A.pl + (int64_t)(head / A.rp) * A.ph + n0 + tj;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (tj + j < nv) dot += (LinDot<IT>)r[j] * (LinDot<IT>)to_f<IT>(p[j]);
            }
          }
          if (A.dot) {
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
            if (tid % 16 == 0 && t < P.seqlen)
              reinterpret_cast<LinDot<IT>*>(A.dot)[(((int64_t)tile * P.batch + b) * P.heads + head) * P.seqlen + t] = dot;
          }
        }
      }
    }
    // H <- e^T H + sum_j w_j k_j v_j^T, R x 4 entries a thread: the first group's part of it while the second
    // writes the outputs; a state alone is shared evenly
    constexpr int R = STATE_ONLY && DMAX == 64 ? 4 : 8;
    const int hi = R == 4 ? tid / 16 * 4 : ti + (second ? 64 : 0);
    if (hi < dk) {
      const float d = expf((float)S.total);
      float h[R][4];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(&S.h[hi + i][tj]);
        h[i][0] = d * x.x, h[i][1] = d * x.y, h[i][2] = d * x.z, h[i][3] = d * x.w;
      }
      for (int n = 0; n < m; n += 4) {
        float4 y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[r] = *reinterpret_cast<const float4*>(&S.v[n + r][tj]);
          const float w = S.w_upd[n + r];
          y[r].x *= w, y[r].y *= w, y[r].z *= w, y[r].w *= w;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(&S.kt[hi + i][n]);
          const float xa[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            h[i][0] = fmaf(xa[r], y[r].x, h[i][0]);
            h[i][1] = fmaf(xa[r], y[r].y, h[i][1]);
            h[i][2] = fmaf(xa[r], y[r].z, h[i][2]);
            h[i][3] = fmaf(xa[r], y[r].w, h[i][3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
        *reinterpret_cast<float4*>(&S.h[hi + i][tj]) = make_float4(h[i][0], h[i][1], h[i][2], h[i][3]);
    }
  }
  __syncthreads();
  if (STATE_ONLY) {
    for (int e = tid; e < dk * nv; e += kLsThreads) {
      const int i = e / nv, j = e % nv;
      A.sum[((int64_t)bh * P.segs + seg) * block + (int64_t)i * dv + n0 + j] = S.h[i][j];
    }
    if (tid == 0 && tile == 0)  // the same value from every pass of a direction
      P.seg_decay[((int64_t)A.reverse * P.batch * P.heads + bh) * P.segs + seg] = (float)seg_total;
  } else if (A.s_out && seg == P.segs - 1) {
    for (int e = tid; e < dk * nv; e += kLsThreads) {
      const int i = e / nv, j = e % nv;
      A.s_out[bh * block + (int64_t)i * A.s_row + (int64_t)(n0 + j) * A.s_col] = A.s_out_scale * S.h[i][j];
    }
  }
}

// The segments' own states -> the state before each segment, in place: a thread an entry, its segments in
// order, 8 loads under way at a time.  About 3 us; folded by the main pass itself, each CTA the segments before
// its own, the same states took 75 us of it.
__global__ void __launch_bounds__(256) linear_fold_kernel(const __grid_constant__ LinK P) {
  griddep_launch_dependents();  // the main pass's first segments need no fold; the others wait for it
  griddep_wait();
  const LinPass& A = P.pass[blockIdx.z];
  const int64_t block = (int64_t)A.dk * A.dv, bh = blockIdx.y;
  __shared__ float decay[32];
  if (threadIdx.x < P.segs - 1)
    decay[threadIdx.x] = expf(P.seg_decay[((int64_t)A.reverse * P.batch * P.heads + bh) * P.segs + threadIdx.x]);
  __syncthreads();
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= block) return;
  float s = A.s_in ? A.s_in_scale * A.s_in[bh * block + e / A.dv * A.s_row + e % A.dv * A.s_col] : 0.f;
  float* at = A.sum + bh * P.segs * block + e;
  for (int q0 = 0; q0 < P.segs; q0 += 8) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = q0 + u < P.segs - 1 ? at[(q0 + u) * block] : 0.f;  // the last one's own is not needed
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (q0 + u < P.segs) {
        at[(q0 + u) * block] = s;
        if (q0 + u < P.segs - 1) s = fmaf(decay[q0 + u], s, x[u]);
      }
  }
}

// ---------------------------------------------------------------------------------- gradient tails
// Gradients of shared heads: out[b, t, kh, d] = sum over the group's heads of parts[b, t, h, d]
// (fp32, contiguous), in a fixed order, rounded once.  Bound by the parts' traffic: 4 x 1999 tokens of 16 heads
// in groups of 4 (131 MB of parts, 16 MB out) take 30 us, 75 % of the copy rate.
struct LinGroupK {
  const float* parts[2];
  void* out[2];
  int64_t ob[2], ol[2], oh[2];
  int batch, seqlen, key_heads, rep, dim;
};

template <typename IT, int VW>
__global__ void __launch_bounds__(256) linear_group_sum_kernel(const __grid_constant__ LinGroupK P) {
  const int which = blockIdx.y, nd = P.dim / VW;
  const int64_t n = (int64_t)P.batch * P.seqlen * P.key_heads * nd;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (int64_t)gridDim.x * blockDim.x) {
    const int d = (int)(e % nd) * VW;
    const int64_t r = e / nd;  // (b, t, kh)
    const float* src = P.parts[which] + (r * P.rep) * P.dim + d;
    float s[VW] = {};
#pragma unroll 4
    for (int i = 0; i < P.rep; ++i) {
      float x[VW];
      if constexpr (VW == 4) {
        const float4 q = *reinterpret_cast<const float4*>(src + (int64_t)i * P.dim);
        x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
      } else {
        x[0] = src[(int64_t)i * P.dim];
      }
#pragma unroll
      for (int k = 0; k < VW; ++k) s[k] += x[k];
    }
    const int kh = (int)(r % P.key_heads);
    const int64_t bt = r / P.key_heads;
    IT* out = static_cast<IT*>(P.out[which]) + (bt / P.seqlen) * P.ob[which] + (bt % P.seqlen) * P.ol[which] + kh * P.oh[which] + d;
#pragma unroll
    for (int k = 0; k < VW; ++k) out[k] = from_f<IT>(s[k]);
  }
}

// dg_t = sum_{i >= t} (q_i . dq_i - k_i . dk_i) + <dS_last, S_last>, summed from the last token.  One CTA per
// (b, h), 512 tokens a step; for a decay per head one CTA per head, which sums over its rows and tokens in a
// fixed order.  Bound by the latency of its steps: 14 us for 192 rows of 2048 tokens (5 MB).
struct LinDecayK {
  const void *xq, *yk;   // [tile][b][h][t], the kernel's T
  int tq, tk;            // tiles of each
  const float *d_last, *last;  // nullable (b, h, dk * dv)
  int64_t block;
  const void* g;
  void* dg;
  int g_f32, per_head, g_bf16;
  int64_t gb, gl, gh;
  const int* lens;
  int batch, seqlen, heads;
};

constexpr int kLdThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kLdThreads) linear_decay_grad_kernel(const __grid_constant__ LinDecayK P) {
  __shared__ double part[kLdThreads / 32];
  __shared__ T part_t[2][kLdThreads / 32];
  __shared__ double carry_s;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int head = P.per_head ? blockIdx.x : blockIdx.x % P.heads;
  const int b0 = P.per_head ? 0 : blockIdx.x / P.heads, b1 = P.per_head ? P.batch : b0 + 1;
  const int64_t bhl = (int64_t)P.batch * P.heads * P.seqlen;
  double sum = 0.0;  // per head: this thread's part of the total
  auto store = [&](int64_t at, float x) {
    if (P.g_f32) static_cast<float*>(P.dg)[at] = x;
    else if (P.g_bf16) static_cast<__nv_bfloat16*>(P.dg)[at] = from_f<__nv_bfloat16>(x);
    else static_cast<__half*>(P.dg)[at] = from_f<__half>(x);
  };
  for (int b = b0; b < b1; ++b) {
    const int64_t bh = (int64_t)b * P.heads + head;
    const int len = P.lens ? max(0, min(P.lens[b], P.seqlen)) : P.seqlen;
    double x = 0.0;
    if (P.d_last)
      for (int64_t e = tid; e < P.block; e += kLdThreads)
        x += (double)P.d_last[bh * P.block + e] * (double)P.last[bh * P.block + e];
    __syncthreads();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) part[wid] = x;
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int i = 0; i < kLdThreads / 32; ++i) s += part[i];
      carry_s = s;
    }
    __syncthreads();
    double carry = carry_s;
    // thread i holds token end - 1 - i, so a prefix over threads is a suffix over tokens; the next tokens'
    // loads are under way while these are summed
    T xn = 0;
    float gn = 0.f;
    auto load = [&](int end) {
      const int t = end - 1 - tid;
      xn = 0, gn = 0.f;
      if (t < 0) return;
      const int64_t at = (int64_t)b * P.gb + (int64_t)t * P.gl + (int64_t)head * P.gh;
      if (P.g_f32) gn = static_cast<const float*>(P.g)[at];
      else if (P.g_bf16) gn = to_f<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(P.g)[at]);
      else gn = to_f<__half>(static_cast<const __half*>(P.g)[at]);
      if (t >= len) return;
      T s = 0, r = 0;  // one or two tiles each
      for (int i = 0; i < P.tq; ++i) s += static_cast<const T*>(P.xq)[i * bhl + bh * P.seqlen + t];
      for (int i = 0; i < P.tk; ++i) r += static_cast<const T*>(P.yk)[i * bhl + bh * P.seqlen + t];
      xn = s - r;
    };
    load(P.seqlen);
    for (int end = P.seqlen; end > 0; end -= kLdThreads) {
      const int t = end - 1 - tid;
      const float g = gn;
      T d = xn;  // a step's 512 tokens in T, the steps in 64 bits
      load(end - kLdThreads);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, d, o);
        if (lane >= o) d += u;
      }
      const int slot = (end / kLdThreads) & 1;
      if (lane == 31) part_t[slot][wid] = d;
      __syncthreads();
      const T w = lane < kLdThreads / 32 ? part_t[slot][lane] : T(0);
      T before = lane < wid ? w : T(0), all = w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
      }
      if (t >= 0) {
        // a reset passes nothing from before the token, and behind the row's end there is nothing
        const double r = t >= len || g < kLinZeroBelow ? 0.0 : carry + (double)(before + d);
        if (P.per_head) sum += r;
        else store(((int64_t)b * P.seqlen + t) * P.heads + head, (float)r);
      }
      carry += (double)all;
    }
  }
  if (P.per_head) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) part[wid] = sum;
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int i = 0; i < kLdThreads / 32; ++i) s += part[i];
      store(head, (float)s);
    }
  }
}

// ------------------------------------------------------------------------------------ single token
// S <- e^g S + k v^T, o = scale q S.  The state is read and written once, a float4 a lane: LPR lanes hold a
// row of the state (8, 16 or 32 for up to 32, 64 or 128 columns), so that narrow heads fill their warps too.
// Bound by the state's traffic: 64 x 40 heads of 128 x 128 move 337 MB in 55 us with the launch, 93 % of the
// copy rate.
struct LinStepK {
  ss_linear_step_args a;
  int vec;
};

constexpr int kLstWarps = 8;

template <typename IT, int LPR>
__global__ void __launch_bounds__(32 * kLstWarps) linear_step_kernel(const __grid_constant__ LinStepK P) {
  const ss_linear_step_args& a = P.a;
  __shared__ float4 red[kLstWarps][32];
  __shared__ float qs[kLinMaxDim], ks[kLinMaxDim];
  const int bh = blockIdx.x, b = bh / a.heads, head = bh % a.heads;
  const int dk = a.key_dim, dv = a.value_dim;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int kh = head / (a.heads / a.key_heads);
  for (int d = threadIdx.x; d < dk; d += blockDim.x) {
    qs[d] = to_f<IT>(static_cast<const IT*>(a.q)[(int64_t)b * a.q_batch_stride + (int64_t)kh * a.q_head_stride + d]);
    ks[d] = to_f<IT>(static_cast<const IT*>(a.k)[(int64_t)b * a.k_batch_stride + (int64_t)kh * a.k_head_stride + d]);
  }
  const int64_t gat = (int64_t)b * a.decay_batch_stride + (int64_t)head * a.decay_head_stride;
  const float g = a.decay_dtype == SS_F32 ? static_cast<const float*>(a.log_decay)[gat]
                                          : to_f<IT>(static_cast<const IT*>(a.log_decay)[gat]);
  const float decay = expf(g);
  const int n0 = lane % LPR * 4, sub = lane / LPR;
  constexpr int step = 32 / LPR * kLstWarps;
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = n0 + j < dv ? to_f<IT>(static_cast<const IT*>(a.v)[(int64_t)b * a.v_batch_stride +
                                                             (int64_t)head * a.v_head_stride + n0 + j]) : 0.f;
  __syncthreads();
  float* st = a.state + (int64_t)b * a.state_batch_stride + (int64_t)head * dk * dv;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  if (n0 < dv) {
    constexpr int U = 8;  // rows of a lane under way at once
    for (int d0 = wid * (32 / LPR) + sub; d0 < dk; d0 += U * step) {
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int d = d0 + u * step;
        const float* row = st + (int64_t)d * dv + n0;
        if (P.vec) {
          if (d < dk) x[u] = *reinterpret_cast<const float4*>(row);
        } else {
          float* e = reinterpret_cast<float*>(&x[u]);
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = d < dk && n0 + j < dv ? row[j] : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int d = d0 + u * step;
        if (d >= dk) break;
        float* row = st + (int64_t)d * dv + n0;
        float* s = reinterpret_cast<float*>(&x[u]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[j] = fmaf(decay, s[j], ks[d] * v[j]);
          o[j] = fmaf(qs[d], s[j], o[j]);
        }
        if (P.vec) {
          *reinterpret_cast<float4*>(row) = x[u];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n0 + j < dv) row[j] = s[j];
        }
      }
    }
  }
  red[wid][lane] = make_float4(o[0], o[1], o[2], o[3]);
  __syncthreads();
  if (wid == 0 && lane < LPR) {
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = lane; i < 32 * kLstWarps; i += LPR) {  // the rows' slices in a fixed order
      const float4 x = red[i >> 5][i & 31];
      r[0] += x.x, r[1] += x.y, r[2] += x.z, r[3] += x.w;
    }
    IT* out = static_cast<IT*>(a.o) + (int64_t)b * a.o_batch_stride + (int64_t)head * a.o_head_stride;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n0 + j < dv) out[n0 + j] = from_f<IT>(a.scale * r[j]);
  }
}

}  // namespace ssb
