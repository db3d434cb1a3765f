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
// every tensor moves once.  A row belongs to WPR warps, each lane holding NV groups of 4 values of every
// tensor (8 bytes of a 16-bit type, 16 of fp32): up to 12 values a lane where 8 warps hold the row so, where the
// 24 of one warp to a row of 768 spilled (163 us a pass over 16384 rows).  128 registers hold the backward's
// rows, weights and column sums then for gated 16-bit rows of two warps and more and for fp32 rows without a gate
// (nothing or a few bytes spilled); gated fp32 rows spill about 300 bytes a thread, gated 16-bit rows of one warp
// 200, and rows longer than 8 warps of 12 values (16 - 32 values a lane) up to 2 KB.  A row's warps meet at a barrier of their own.  A lane's columns are the same for all its
// rows: their weights are loaded once, with the first row, and in the backward their two sums stay in
// registers over the rows of a persistent CTA; the CTAs' sums meet in a second small kernel (4 us) in a fixed
// order, so the gradients of the weights do not vary between runs.
// Measured (kernels, cold L2; shares of the copy rate), forward and backward:
//   16384 x 768 bf16, gated       28 us 69 %    44 us 70 %  (65 us with each row loaded when its turn comes)
//   4099 x 2560 fp32              32 us 81 %    45 us 86 %  (51 us)
//   8192 x 768 fp32, gated        26 us 74 %    52 us 60 %
//   32768 x 384 bf16, gated       28 us 69 %    65 us 47 %
//   2048 x 8192 bf16, gated       60 us 43 %   185 us 22 %
//   2048 x 8192 fp32, gated       72 us 72 %   323 us 25 %
// 69 - 70 % is latency: 24 warps an SM wait for their rows half of the time in the forward (16 in the backward,
// which issues in 60 % of its cycles); below 60 % it is the spills.
#pragma once
#include "ss_norm.cuh"

namespace ssb {

constexpr int kBnWarps = 8;

enum { kActNone = 0, kActSilu = 1, kActSigmoid = 2 };

struct BlockNormK {
  ss_block_norm_args a;
  int vec, wvec;  // rows, weights: whole 16-byte vectors
};

struct BlockNormBwdK {
  ss_block_norm_bwd_args a;
  int vec, wvec;
};

// act(z) from the sigmoid of z, and its slope
__device__ __forceinline__ float act_of(int act, float z, float sg) {
  return act == kActSilu ? z * sg : act == kActSigmoid ? sg : z;
}
__device__ __forceinline__ float slope_of(int act, float z, float sg) {
  return act == kActSilu ? sg * fmaf(z, 1.f - sg, 1.f) : act == kActSigmoid ? sg * (1.f - sg) : 1.f;
}

constexpr int kBv = 4;  // values of a vector

// kBv weights of the columns from e0 on; `none` where there are no weights, 0 beyond the row
__device__ __forceinline__ void load_weights(float (&w)[kBv], const float* p, int e0, int dim, float ofs, float none,
                                             bool vec) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < kBv; ++k) w[k] = none;
  } else if (vec) {
    const float4 x = e0 < dim ? __ldg(reinterpret_cast<const float4*>(p + e0)) : make_float4(0.f, 0.f, 0.f, 0.f);
    w[0] = x.x + ofs, w[1] = x.y + ofs, w[2] = x.z + ofs, w[3] = x.w + ofs;
  } else {
#pragma unroll
    for (int k = 0; k < kBv; ++k) w[k] = e0 + k < dim ? p[e0 + k] + ofs : 0.f;
  }
}

template <typename IT> struct BnVec { using T = uint2; };
template <> struct BnVec<float> { using T = uint4; };

// sum over a row's WPR warps; `slot` alternates between uses, so that one barrier a sum is enough
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[kBnWarps], int slot) {
  v = warp_sum(v);
  if constexpr (WPR > 1) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, w0 = wid / WPR * WPR;
    if (lane == 0) red[slot][wid] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + wid / WPR), "n"(32 * WPR) : "memory");
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) v += red[slot][w0 + i];
  }
  return v;
}

// a lane's first element of vector j of its row: warp `part` of WPR
template <int WPR>
__device__ __forceinline__ int bn_at(int j, int part, int lane) { return ((j * WPR + part) * 32 + lane) * kBv; }

// streaming load of a vector, zeros where `on` is false; predicated inside, since a branch around the load
// would wait for it before the next one is issued
__device__ __forceinline__ uint2 ld_stream(const uint2* p, bool on) {
  uint2 r;
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %3, 0;\n mov.u32 %0, 0;\n mov.u32 %1, 0;\n"
               " @p ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n}\n"
               : "=&r"(r.x), "=&r"(r.y) : "l"(p), "r"((uint32_t)on));
  return r;
}
__device__ __forceinline__ uint4 ld_stream(const uint4* p, bool on) {
  uint4 r;
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %5, 0;\n mov.u32 %0, 0;\n mov.u32 %1, 0;\n mov.u32 %2, 0;\n mov.u32 %3, 0;\n"
               " @p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n}\n"
               : "=&r"(r.x), "=&r"(r.y), "=&r"(r.z), "=&r"(r.w) : "l"(p), "r"((uint32_t)on));
  return r;
}

template <typename IT, int NV, int WPR>
__device__ __forceinline__ void bn_load(typename BnVec<IT>::T (&q)[NV], const IT* row, int dim, int part, int lane, bool vec) {
  using V = typename BnVec<IT>::T;
  if (vec) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = bn_at<WPR>(j, part, lane);
      q[j] = ld_stream(reinterpret_cast<const V*>(row + e0), e0 < dim);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = bn_at<WPR>(j, part, lane);
      union { V u; IT e[kBv]; } pk;
#pragma unroll
      for (int k = 0; k < kBv; ++k) pk.e[k] = (e0 + k < dim) ? row[e0 + k] : zero_v<IT>();
      q[j] = pk.u;
    }
  }
}

// asynchronous copy of a vector into shared memory, zeros where `on` is false
template <typename V>
__device__ __forceinline__ void bn_fetch(V* to, const void* from, bool on) {
  if constexpr (sizeof(V) == 8)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(on ? 8 : 0) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(on ? 16 : 0) : "memory");
}

template <typename IT>
__device__ __forceinline__ void bn_store(IT* row, int e0, const float (&v)[kBv], int dim, bool vec) {
  using V = typename BnVec<IT>::T;
  if (e0 >= dim) return;
  if (vec) {
    union { V u; IT e[kBv]; } pk;
#pragma unroll
    for (int k = 0; k < kBv; ++k) pk.e[k] = from_f<IT>(v[k]);
    *reinterpret_cast<V*>(row + e0) = pk.u;
  } else {
#pragma unroll
    for (int k = 0; k < kBv; ++k)
      if (e0 + k < dim) row[e0 + k] = from_f<IT>(v[k]);
  }
}

template <typename IT>
__device__ __forceinline__ void unpack(float (&v)[kBv], const typename BnVec<IT>::T& q) {
  union { typename BnVec<IT>::T u; IT e[kBv]; } pk;
  pk.u = q;
#pragma unroll
  for (int k = 0; k < kBv; ++k) v[k] = to_f<IT>(pk.e[k]);
}

// MODE: 0 any call; 1 both norms, whole vectors (and dh in the backward), no gate; 2 the same with a SiLU
// gate.  The common calls know at compile time what the others branch on for every vector (16384 rows of 768
// with a gate, bf16: forward 45 -> 28 us, backward 100 -> 65 us, and 43 with the rows fetched ahead).
enum { kBnAny = 0, kBnPlain = 1, kBnGated = 2 };

template <typename IT, int NV, int WPR, int MODE>
__global__ void __launch_bounds__(32 * kBnWarps) block_norm_fwd_kernel(const __grid_constant__ BlockNormK P) {
  using V = typename BnVec<IT>::T;
  constexpr int RPC = kBnWarps / WPR;  // rows of a CTA at a time
  __shared__ float red[2][kBnWarps];
  const ss_block_norm_args& a = P.a;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, part = wid % WPR;
  const int dim = a.dim;
  const bool gate = MODE ? MODE == kBnGated : a.gate != nullptr, post = MODE || a.post_weight != nullptr,
             pre = MODE || a.pre_weight != nullptr, vec = MODE || P.vec, wvec = MODE || P.wvec;
  const int act = MODE ? (int)kActSilu : a.activation;
  const float ofs = a.unit_offset ? 1.f : 0.f, inv = 1.f / (float)dim;
  float w[NV][kBv], wn[NV][kBv];  // s (1 + w_post), 1 + w_pre
  for (int64_t first = (int64_t)blockIdx.x * RPC + wid / WPR, row = first; row < a.rows; row += (int64_t)gridDim.x * RPC) {
    V yq[NV], rq[NV], zq[NV];
    bn_load<IT, NV, WPR>(yq, (const IT*)a.y + row * a.y_row_stride, dim, part, lane, vec);
    bn_load<IT, NV, WPR>(rq, (const IT*)a.residual + row * a.residual_row_stride, dim, part, lane, vec);
    if (gate) bn_load<IT, NV, WPR>(zq, (const IT*)a.gate + row * a.gate_row_stride, dim, part, lane, vec);
    if (row == first) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = bn_at<WPR>(j, part, lane);
        float sc[kBv];
        load_weights(w[j], a.post_weight, e0, dim, ofs, 1.f, wvec);
        load_weights(sc, a.scale, e0, dim, 0.f, a.scale_const, wvec);
        load_weights(wn[j], a.pre_weight, e0, dim, ofs, 1.f, wvec);
#pragma unroll
        for (int k = 0; k < kBv; ++k) w[j][k] *= sc[k];
      }
    }
    float h[NV][kBv];
    float ss = 0.f, ry = 1.f;
    if (post) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float y[kBv];
        unpack<IT>(y, yq[j]);
#pragma unroll
        for (int k = 0; k < kBv; ++k) ss = fmaf(y[k], y[k], ss);
      }
      ry = rsqrtf(fmaf(row_sum<WPR>(ss, red, 0), inv, a.eps));
    }
    ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float y[kBv], z[kBv];
      unpack<IT>(y, yq[j]);
      unpack<IT>(h[j], rq[j]);
      if (gate) unpack<IT>(z, zq[j]);
#pragma unroll
      for (int k = 0; k < kBv; ++k) {
        float u = y[k] * ry * w[j][k];
        if (gate) u *= act_of(act, z[k], sigmoid_fast(z[k]));
        h[j][k] += u;
        ss = fmaf(h[j][k], h[j][k], ss);
      }
      bn_store<IT>((IT*)a.h + row * a.h_row_stride, bn_at<WPR>(j, part, lane), h[j], dim, vec);
    }
    float rh = 0.f;
    if (pre) {
      rh = rsqrtf(fmaf(row_sum<WPR>(ss, red, 1), inv, a.pre_eps));
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int k = 0; k < kBv; ++k) h[j][k] *= rh * wn[j][k];
        bn_store<IT>((IT*)a.x + row * a.x_row_stride, bn_at<WPR>(j, part, lane), h[j], dim, vec);
      }
    }
    if (a.rstd && part == 0 && lane == 0) *reinterpret_cast<float2*>(a.rstd + 2 * row) = make_float2(ry, rh);
    // one sum a row: without the other's barrier the next row's write could meet this row's reads
    if (WPR > 1 && !(post && pre)) asm volatile("bar.sync %0, %1;" ::"r"(1 + wid / WPR), "n"(32 * WPR) : "memory");
  }
}

template <typename IT, int NV, int WPR, int MODE>
__global__ void __launch_bounds__(32 * kBnWarps, 2)
    block_norm_bwd_kernel(const __grid_constant__ BlockNormBwdK P) {
  using V = typename BnVec<IT>::T;
  constexpr int RPC = kBnWarps / WPR;
  extern __shared__ __align__(16) float sums[];  // a column sum of the CTA's rows
  __shared__ float red[2][kBnWarps];
  const ss_block_norm_args& a = P.a.f;
  const ss_block_norm_bwd_args& g = P.a;
  const bool has_dh = MODE || g.dh != nullptr;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, part = wid % WPR;
  const int dim = a.dim;
  const bool gate = MODE ? MODE == kBnGated : a.gate != nullptr, post = MODE || a.post_weight != nullptr,
             pre = MODE || a.pre_weight != nullptr, vec = MODE || P.vec, wvec = MODE || P.wvec;
  const int act = MODE ? (int)kActSilu : a.activation;
  const float ofs = a.unit_offset ? 1.f : 0.f, inv = 1.f / (float)dim;
  float w[NV][kBv], wn[NV][kBv], sx[NV][kBv], sp[NV][kBv];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = bn_at<WPR>(j, part, lane);
    float sc[kBv];
    load_weights(w[j], a.post_weight, e0, dim, ofs, 1.f, wvec);
    load_weights(sc, a.scale, e0, dim, 0.f, a.scale_const, wvec);
    load_weights(wn[j], a.pre_weight, e0, dim, ofs, 1.f, wvec);
#pragma unroll
    for (int k = 0; k < kBv; ++k) w[j][k] *= sc[k], sx[j][k] = sp[j][k] = 0.f;
  }
  // The common calls fetch the next row while this one is computed: a thread's own vectors, into its own room.
  // 16-bit rows have two rooms and are read again for each use (63 us with one room, from registers that spill);
  // fp32 rows, with room for one, move into registers
  constexpr bool kRooms = MODE != 0 && sizeof(IT) == 2;
  constexpr int kTensors = MODE == kBnGated ? 5 : 4;
  V* room = reinterpret_cast<V*>(sums + NV * WPR * 32 * kBv) + threadIdx.x;
  V *here = room, *there = room + (kRooms ? kTensors * NV * 32 * kBnWarps : 0);
  auto slot = [&](V* in, int t, int j) { return in + (t * NV + j) * 32 * kBnWarps; };
  auto fetch = [&](V* in, int64_t row) {
    auto one = [&](int t, const void* p, int64_t stride) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = bn_at<WPR>(j, part, lane);
        bn_fetch(slot(in, t, j), (const IT*)p + row * stride + (e0 < dim ? e0 : 0), e0 < dim);
      }
    };
    if (row < a.rows) {
      one(0, a.y, a.y_row_stride);
      one(1, a.residual, a.residual_row_stride);
      one(2, g.dx, g.dx_row_stride);
      one(3, g.dh, g.dh_row_stride);
      if (gate) one(4, a.gate, a.gate_row_stride);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int64_t first = (int64_t)blockIdx.x * RPC + wid / WPR, hop = (int64_t)gridDim.x * RPC;
  if constexpr (MODE != 0) fetch(here, first);
  for (int64_t row = first; row < a.rows; row += hop) {
    V yq[NV], rq[NV], zq[NV], xq[NV], hq[NV];
    const float2 rr = *reinterpret_cast<const float2*>(a.rstd + 2 * row);
    if constexpr (kRooms) {
      fetch(there, row + hop);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else if constexpr (MODE != 0) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        yq[j] = *slot(here, 0, j), rq[j] = *slot(here, 1, j), xq[j] = *slot(here, 2, j), hq[j] = *slot(here, 3, j);
        if (gate) zq[j] = *slot(here, 4, j);
      }
      fetch(here, row + hop);
    } else {
      bn_load<IT, NV, WPR>(yq, (const IT*)a.y + row * a.y_row_stride, dim, part, lane, vec);
      bn_load<IT, NV, WPR>(rq, (const IT*)a.residual + row * a.residual_row_stride, dim, part, lane, vec);
      if (gate) bn_load<IT, NV, WPR>(zq, (const IT*)a.gate + row * a.gate_row_stride, dim, part, lane, vec);
      if (pre) bn_load<IT, NV, WPR>(xq, (const IT*)g.dx + row * g.dx_row_stride, dim, part, lane, vec);
      if (has_dh) bn_load<IT, NV, WPR>(hq, (const IT*)g.dh + row * g.dh_row_stride, dim, part, lane, vec);
    }
    const float ry = rr.x, rh = rr.y;
    auto take = [&](float (&v)[kBv], int t, const V& q, int j) {
      if constexpr (kRooms) unpack<IT>(v, *slot(here, t, j));
      else unpack<IT>(v, q);
    };
    float h[NV][kBv];  // h, then u
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float y[kBv], z[kBv], d[kBv];
      take(y, 0, yq[j], j);
      take(h[j], 1, rq[j], j);
      if (gate) take(z, 4, zq[j], j);
      if (pre) take(d, 2, xq[j], j);
#pragma unroll
      for (int k = 0; k < kBv; ++k) {
        float u = y[k] * ry * w[j][k];
        if (gate) u *= act_of(act, z[k], sigmoid_fast(z[k]));
        h[j][k] += u;
        if (pre) {
          dot = fmaf(d[k] * wn[j][k], h[j][k], dot);
          sp[j][k] = fmaf(d[k], h[j][k] * rh, sp[j][k]);
        }
      }
    }
    float c = 0.f;
    if (pre) c = row_sum<WPR>(dot, red, 0) * inv * rh * rh;
    dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float y[kBv], z[kBv], d[kBv], gh[kBv], dz[kBv];
      take(y, 0, yq[j], j);
      if (gate) take(z, 4, zq[j], j);
      if (pre) take(d, 2, xq[j], j);
      if (has_dh) take(gh, 3, hq[j], j);
#pragma unroll
      for (int k = 0; k < kBv; ++k) {
        if (!has_dh) gh[k] = 0.f;
        if (pre) gh[k] = fmaf(rh, fmaf(d[k], wn[j][k], -h[j][k] * c), gh[k]);
        const float n = y[k] * ry;
        float f = 1.f;
        if (gate) {
          const float sg = sigmoid_fast(z[k]);
          f = act_of(act, z[k], sg);
          dz[k] = gh[k] * w[j][k] * n * slope_of(act, z[k], sg);
        }
        sx[j][k] = fmaf(gh[k] * f, n, sx[j][k]);
        h[j][k] = gh[k] * w[j][k] * f;
        dot = fmaf(h[j][k], n, dot);
      }
      const int e0 = bn_at<WPR>(j, part, lane);
      bn_store<IT>((IT*)g.dresidual + row * g.dresidual_row_stride, e0, gh, dim, vec);
      if (gate) bn_store<IT>((IT*)g.dgate + row * g.dgate_row_stride, e0, dz, dim, vec);
    }
    float m = 0.f;
    if (post) m = row_sum<WPR>(dot, red, 1) * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (post) {
        float y[kBv];
        take(y, 0, yq[j], j);
#pragma unroll
        for (int k = 0; k < kBv; ++k) h[j][k] = ry * (h[j][k] - y[k] * ry * m);
      }
      bn_store<IT>((IT*)g.dy + row * g.dy_row_stride, bn_at<WPR>(j, part, lane), h[j], dim, vec);
    }
    if constexpr (kRooms) {
      V* t = here;
      here = there, there = t;
    }
    if (WPR > 1 && !(post && pre)) asm volatile("bar.sync %0, %1;" ::"r"(1 + wid / WPR), "n"(32 * WPR) : "memory");
  }
  // this CTA's column sums: its row groups in order, then to the workspace
  __syncthreads();
  float* out = g.work + (int64_t)blockIdx.x * 2 * dim;
  for (int s = 0; s < 2; ++s) {
    for (int r = 0; r < RPC; ++r) {
      if (wid / WPR == r) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const float4 v = s ? make_float4(sp[j][0], sp[j][1], sp[j][2], sp[j][3])
                             : make_float4(sx[j][0], sx[j][1], sx[j][2], sx[j][3]);
          float4* to = reinterpret_cast<float4*>(sums + bn_at<WPR>(j, part, lane));
          const float4 x = r ? *to : make_float4(0.f, 0.f, 0.f, 0.f);
          *to = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
        }
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < dim; e += blockDim.x) out[s * dim + e] = sums[e];
    __syncthreads();
  }
}

// Column sums over the CTAs' partial sums: 32 columns and 32 slices of the CTAs per block, added in
// a fixed order.
__global__ void __launch_bounds__(1024) block_norm_cols_kernel(const float* work, int parts, int dim,
                                                              const float* post_weight, const float* scale,
                                                              float scale_const, float ofs, float* dpost, float* dpre,
                                                              float* dscale) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane, which = blockIdx.y;
  float s = 0.f;
  if (col < dim)
    for (int i = wid; i < parts; i += 32) s += work[((int64_t)i * 2 + which) * dim + col];
  red[wid][lane] = s;
  __syncthreads();
  if (wid == 0 && col < dim) {
#pragma unroll
    for (int i = 1; i < 32; ++i) s += red[i][lane];
    if (which) {
      if (dpre) dpre[col] = s;
    } else {
      if (dpost) dpost[col] = s * (scale ? scale[col] : scale_const);
      if (dscale) dscale[col] = s * (post_weight ? post_weight[col] + ofs : 1.f);
    }
  }
}

}  // namespace ssb
