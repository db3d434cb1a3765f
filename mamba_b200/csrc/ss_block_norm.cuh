// The norms before and after a block, with the block's gate and the residual scale, in one pass:
//
//   n = y * rsqrt(mean(y^2) + eps)                    (n = y without a post weight)
//   h = residual + s * act(z) * (1 + w_post) * n      the next residual stream
//   x = h * rsqrt(mean(h^2) + pre_eps) * (1 + w_pre)      the next block's input
//
// All in fp32 from the inputs, each output rounded once (x comes from the unrounded h).
// Backward, with t = dx (1 + w_pre), r_y and r_h the two reciprocal roots from the forward:
//
//   gh = dh + r_h (t - h r_h^2 mean(t h)) = dresidual       h recomputed from y, z, residual
//   u  = gh s act(z) (1 + w_post);   dy = r_y (u - n mean(u n));   dz = gh s (1 + w_post) n act'(z)
//   X  = sum over rows of gh act(z) n:   dw_post = s X,   ds = (1 + w_post) X;   dw_pre = sum of dx h r_h
//
// Bound by the memory traffic: the rows stay in registers between the statistics and their use, so
// every tensor moves once.  A row belongs to WPR warps (one up to 768 ... 1024 16-bit values, so
// that its two reductions need no barrier), each lane holding NV 16-byte vectors of every tensor;
// CTAs are persistent and keep the columns' factors in shared memory, and in the backward the two
// column sums in registers until a CTA's rows are done.  The CTAs' sums meet in a second small
// kernel in a fixed order, so the gradients of the weights do not vary between runs.
#pragma once
#include "ss_norm.cuh"

namespace ssb {

constexpr int kBnWarps = 8;

enum { kActNone = 0, kActSilu = 1, kActSigmoid = 2 };

struct BlockNormK {
  ss_block_norm_args a;
  int vec;
};

struct BlockNormBwdK {
  ss_block_norm_bwd_args a;
  int vec;
};

// act(z) and its slope
__device__ __forceinline__ void gate_act(int act, float z, float& f, float& df) {
  const float sg = 1.f / (1.f + __expf(-z));
  if (act == kActSilu) {
    f = z * sg;
    df = sg * fmaf(z, 1.f - sg, 1.f);
  } else {
    f = sg;
    df = sg * (1.f - sg);
  }
}

// sum over a row's WPR warps; `slot` alternates between uses so that one barrier a sum is enough
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[kBnWarps], int slot) {
  v = warp_sum(v);
  if constexpr (WPR > 1) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    if (lane == 0) red[slot][wid] = v;
    __syncthreads();
    const int w0 = wid / WPR * WPR;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) v += red[slot][w0 + i];
  }
  return v;
}

// a row's vectors: lane `lane` of warp `part` holds elements ((j * WPR + part) * 32 + lane) * VW + k
template <typename IT, int NV, int WPR>
__device__ __forceinline__ void bn_load(uint4 (&q)[NV], const IT* row, int dim, int part, int lane, bool vec) {
  constexpr int VW = 16 / sizeof(IT);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = ((j * WPR + part) * 32 + lane) * VW;
    if (vec) {
      q[j] = e0 < dim ? ld_stream16(row + e0) : make_uint4(0u, 0u, 0u, 0u);
    } else {
      union { uint4 u; IT e[VW]; } pk;
#pragma unroll
      for (int k = 0; k < VW; ++k) pk.e[k] = (e0 + k < dim) ? row[e0 + k] : zero_v<IT>();
      q[j] = pk.u;
    }
  }
}

template <typename IT>
__device__ __forceinline__ void bn_store(IT* row, int e0, const float (&v)[16 / sizeof(IT)], int dim, bool vec) {
  constexpr int VW = 16 / sizeof(IT);
  if (e0 >= dim) return;
  if (vec) {
    uint4 pk;
    IT* e = reinterpret_cast<IT*>(&pk);
#pragma unroll
    for (int k = 0; k < VW; ++k) e[k] = from_f<IT>(v[k]);
    *reinterpret_cast<uint4*>(row + e0) = pk;
  } else {
#pragma unroll
    for (int k = 0; k < VW; ++k)
      if (e0 + k < dim) row[e0 + k] = from_f<IT>(v[k]);
  }
}

template <typename IT>
__device__ __forceinline__ float lane_of(const uint4& q, int k) {
  return to_f<IT>(reinterpret_cast<const IT*>(&q)[k]);
}

template <typename IT, int NV, int WPR>
__global__ void __launch_bounds__(32 * kBnWarps) block_norm_fwd_kernel(const __grid_constant__ BlockNormK P) {
  constexpr int VW = 16 / sizeof(IT);
  constexpr int LEN = NV * WPR * 32 * VW;
  constexpr int RPC = kBnWarps / WPR;  // rows of a CTA at a time
  extern __shared__ __align__(16) float w_s[];  // [0, LEN): s (1 + w_post); [LEN, 2 LEN): 1 + w_pre
  __shared__ float red[2][kBnWarps];
  const ss_block_norm_args& a = P.a;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, part = wid % WPR;
  const int dim = a.dim;
  const bool gate = a.gate != nullptr, post = a.post_weight != nullptr, pre = a.pre_weight != nullptr;
  const float ofs = a.unit_offset ? 1.f : 0.f, inv = 1.f / (float)dim;
  for (int e = threadIdx.x; e < LEN; e += blockDim.x) {
    const bool on = e < dim;
    w_s[e] = on ? (a.scale ? a.scale[e] : a.scale_const) * (post ? a.post_weight[e] + ofs : 1.f) : 0.f;
    w_s[LEN + e] = on && pre ? a.pre_weight[e] + ofs : 0.f;
  }
  __syncthreads();
  for (int64_t r0 = (int64_t)blockIdx.x * RPC; r0 < a.rows; r0 += (int64_t)gridDim.x * RPC) {
    const int64_t row = r0 + wid / WPR;
    const bool on = row < a.rows;  // the same for the row's warps; idle ones only join the barriers
    uint4 yq[NV], rq[NV], zq[NV];
    float h[NV][VW];
    float ss = 0.f;
    if (on) {
      bn_load<IT, NV, WPR>(yq, (const IT*)a.y + row * a.y_row_stride, dim, part, lane, P.vec);
      bn_load<IT, NV, WPR>(rq, (const IT*)a.residual + row * a.residual_row_stride, dim, part, lane, P.vec);
      if (gate) bn_load<IT, NV, WPR>(zq, (const IT*)a.gate + row * a.gate_row_stride, dim, part, lane, P.vec);
      if (post) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            const float y = lane_of<IT>(yq[j], k);
            ss = fmaf(y, y, ss);
          }
      }
    }
    float ry = 1.f;
    if (post) ry = rsqrtf(fmaf(row_sum<WPR>(ss, red, 0), inv, a.eps));
    ss = 0.f;
    if (on) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = ((j * WPR + part) * 32 + lane) * VW;
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          float u = lane_of<IT>(yq[j], k) * ry * w_s[e0 + k];
          if (gate) {
            float f = lane_of<IT>(zq[j], k), df;
            if (a.activation != kActNone) gate_act(a.activation, f, f, df);
            u *= f;
          }
          h[j][k] = lane_of<IT>(rq[j], k) + u;
          ss = fmaf(h[j][k], h[j][k], ss);
        }
        bn_store<IT>((IT*)a.h + row * a.h_row_stride, e0, h[j], dim, P.vec);
      }
    }
    float rh = 0.f;
    if (pre) {
      rh = rsqrtf(fmaf(row_sum<WPR>(ss, red, 1), inv, a.pre_eps));
      if (on) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int e0 = ((j * WPR + part) * 32 + lane) * VW;
#pragma unroll
          for (int k = 0; k < VW; ++k) h[j][k] *= rh * w_s[LEN + e0 + k];
          bn_store<IT>((IT*)a.x + row * a.x_row_stride, e0, h[j], dim, P.vec);
        }
      }
    }
    if (on && a.rstd && part == 0 && lane == 0) {
      a.rstd[2 * row] = ry;
      a.rstd[2 * row + 1] = rh;
    }
    // one sum a row: without the other's barrier the next row's write could meet this row's reads
    if (WPR > 1 && !(post && pre)) __syncthreads();
  }
}

template <typename IT, int NV, int WPR>
__global__ void __launch_bounds__(32 * kBnWarps) block_norm_bwd_kernel(const __grid_constant__ BlockNormBwdK P) {
  constexpr int VW = 16 / sizeof(IT);
  constexpr int LEN = NV * WPR * 32 * VW;
  constexpr int RPC = kBnWarps / WPR;
  extern __shared__ __align__(16) float w_s[];  // factors as in the forward; then the rows' column sums
  __shared__ float red[2][kBnWarps];
  const ss_block_norm_args& a = P.a.f;
  const ss_block_norm_bwd_args& g = P.a;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, part = wid % WPR;
  const int dim = a.dim;
  const bool gate = a.gate != nullptr, post = a.post_weight != nullptr, pre = a.pre_weight != nullptr;
  const float ofs = a.unit_offset ? 1.f : 0.f, inv = 1.f / (float)dim;
  for (int e = threadIdx.x; e < LEN; e += blockDim.x) {
    const bool on = e < dim;
    w_s[e] = on ? (a.scale ? a.scale[e] : a.scale_const) * (post ? a.post_weight[e] + ofs : 1.f) : 0.f;
    w_s[LEN + e] = on && pre ? a.pre_weight[e] + ofs : 0.f;
  }
  float sx[NV][VW], sp[NV][VW];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VW; ++k) sx[j][k] = sp[j][k] = 0.f;
  __syncthreads();
  for (int64_t r0 = (int64_t)blockIdx.x * RPC; r0 < a.rows; r0 += (int64_t)gridDim.x * RPC) {
    const int64_t row = r0 + wid / WPR;
    const bool on = row < a.rows;
    uint4 yq[NV], rq[NV], zq[NV], xq[NV], hq[NV];
    float ry = 1.f, rh = 0.f;
    float h[NV][VW];  // h, then gh
    float dot = 0.f;
    if (on) {
      bn_load<IT, NV, WPR>(yq, (const IT*)a.y + row * a.y_row_stride, dim, part, lane, P.vec);
      bn_load<IT, NV, WPR>(rq, (const IT*)a.residual + row * a.residual_row_stride, dim, part, lane, P.vec);
      if (gate) bn_load<IT, NV, WPR>(zq, (const IT*)a.gate + row * a.gate_row_stride, dim, part, lane, P.vec);
      if (pre) bn_load<IT, NV, WPR>(xq, (const IT*)g.dx + row * g.dx_row_stride, dim, part, lane, P.vec);
      if (g.dh) bn_load<IT, NV, WPR>(hq, (const IT*)g.dh + row * g.dh_row_stride, dim, part, lane, P.vec);
      ry = a.rstd[2 * row];
      rh = a.rstd[2 * row + 1];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = ((j * WPR + part) * 32 + lane) * VW;
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          float u = lane_of<IT>(yq[j], k) * ry * w_s[e0 + k];
          if (gate) {
            float f = lane_of<IT>(zq[j], k), df;
            if (a.activation != kActNone) gate_act(a.activation, f, f, df);
            u *= f;
          }
          h[j][k] = lane_of<IT>(rq[j], k) + u;
          if (pre) {
            const float d = lane_of<IT>(xq[j], k);
            dot = fmaf(d * w_s[LEN + e0 + k], h[j][k], dot);
            sp[j][k] = fmaf(d, h[j][k] * rh, sp[j][k]);
          }
        }
      }
    }
    float c = 0.f;
    if (pre) c = row_sum<WPR>(dot, red, 0) * inv * rh * rh;
    dot = 0.f;
    if (on) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = ((j * WPR + part) * 32 + lane) * VW;
        float dz[VW];
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          float gh = g.dh ? lane_of<IT>(hq[j], k) : 0.f;
          if (pre) gh = fmaf(rh, fmaf(lane_of<IT>(xq[j], k), w_s[LEN + e0 + k], -h[j][k] * c), gh);
          const float n = lane_of<IT>(yq[j], k) * ry, w = w_s[e0 + k];
          float f = 1.f, df = 1.f;
          if (gate) {
            f = lane_of<IT>(zq[j], k);
            if (a.activation != kActNone) gate_act(a.activation, f, f, df);
          }
          dz[k] = gh * w * n * df;
          sx[j][k] = fmaf(gh * f, n, sx[j][k]);
          dot = fmaf(gh * w * f, n, dot);
          h[j][k] = gh;
        }
        bn_store<IT>((IT*)g.dresidual + row * g.dresidual_row_stride, e0, h[j], dim, P.vec);
        if (gate) bn_store<IT>((IT*)g.dgate + row * g.dgate_row_stride, e0, dz, dim, P.vec);
      }
    }
    float m = 0.f;
    if (post) m = row_sum<WPR>(dot, red, 1) * inv;
    if (on) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = ((j * WPR + part) * 32 + lane) * VW;
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          float f = 1.f, df;
          if (gate) {
            f = lane_of<IT>(zq[j], k);
            if (a.activation != kActNone) gate_act(a.activation, f, f, df);
          }
          const float u = h[j][k] * w_s[e0 + k] * f;
          h[j][k] = post ? ry * (u - lane_of<IT>(yq[j], k) * ry * m) : u;
        }
        bn_store<IT>((IT*)g.dy + row * g.dy_row_stride, e0, h[j], dim, P.vec);
      }
    }
    if (WPR > 1 && !(post && pre)) __syncthreads();
  }
  // this CTA's column sums: its row groups in order, then to the workspace
  __syncthreads();
  float* out = g.work + (int64_t)blockIdx.x * 2 * dim;
  for (int s = 0; s < 2; ++s) {
    for (int r = 0; r < RPC; ++r) {
      if (wid / WPR == r) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            const int e = ((j * WPR + part) * 32 + lane) * VW + k;
            const float v = s ? sp[j][k] : sx[j][k];
            w_s[e] = r ? w_s[e] + v : v;
          }
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < dim; e += blockDim.x) out[s * dim + e] = w_s[e];
    __syncthreads();
  }
}

// Column sums over the CTAs' partial sums: 32 columns and 8 slices of the CTAs per block, added in
// a fixed order.
__global__ void __launch_bounds__(256) block_norm_cols_kernel(const float* work, int parts, int dim,
                                                              const float* post_weight, const float* scale,
                                                              float scale_const, float ofs, float* dpost, float* dpre,
                                                              float* dscale) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane, which = blockIdx.y;
  float s = 0.f;
  if (col < dim)
    for (int i = wid; i < parts; i += 8) s += work[((int64_t)i * 2 + which) * dim + col];
  red[wid][lane] = s;
  __syncthreads();
  if (wid == 0 && col < dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][lane];
    if (which) {
      if (dpre) dpre[col] = s;
    } else {
      if (dpost) dpost[col] = s * (scale ? scale[col] : scale_const);
      if (dscale) dscale[col] = s * (post_weight ? post_weight[col] + ofs : 1.f);
    }
  }
}

}  // namespace ssb
