// One step of beam search: the num_select best continuations over the beams and the vocabulary of
// each batch row, and the reordering of the beams' states.
//
//   cand[w, v] = score[w] + logit[w, v] - log sum_v' e^{logit[w, v']}
//
// Selection, pass 1: CTAs own slices of one beam's vocabulary, read once.  Inside a beam the order
// of the candidates is the order of the logits, so a slice needs only its largest num_select logits
// (the first among equals; where two logits could give one candidate, pass 2 reads the beam again), beside its
// running maximum and sum of exponentials.  A warp keeps the
// best so far sorted over its lanes, as 64-bit keys (the logit's bits mapped to ascending integers,
// then the complement of the index, so one comparison orders both).  Of a batch of 32 logits a lane only those
// are offered that reach the k-th largest of the lanes' maxima (a bound from below) and the list's last: a
// few more than k in the first batch, about k ln 2 each time the number read doubles.
// Pass 2, one CTA per batch row and one warp per beam: slices' sums (in fp64) and keys merged, then
// the beams' lists, compared as fp64 values.  The exponentials, and their sums inside a lane, are fp32 (a lane
// holds up to some 200 terms where a beam is one slice, tens elsewhere), the sums across lanes fp64.  What that
// leaves of the logarithm: an exponential is off by 2^-23 and its argument's rounding, so a row of a few large
// terms by about 1e-7 at most; over many equal rows the roundings average out to 1e-8 - 3e-8, and 1.1e-7 is the
// largest seen.  Two candidates of different beams that are nearer than that may change places against exact
// arithmetic; those of one beam do not, since its logarithm is the same for all.
// Pass 1 takes 31 us for 192 x 50280 fp32 (39 MB, 1.2 TB/s), both 51 us.  Neither memory (15 % of DRAM's rate) nor
// issue slots (53 %) are full: 17 warps an SM wait in turn for fixed latencies, for the loads at the start of each
// batch (nothing is fetched ahead) and for conversions, and the CTAs come in 1.3 waves.
#pragma once
#include "ss_common.cuh"

namespace ssb {

constexpr int kBsThreads = 256;
constexpr int kBsWarps = kBsThreads / 32;
constexpr unsigned kFull = 0xffffffffu;

typedef unsigned long long u64;

// float order as ascending unsigned integers; NaN sorts as -infinity (a beam with one has no valid
// candidate, which the merge sees from its sum)
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as +0
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// the best 32 of a warp, lane i the i-th best (0: none)
struct WarpBest {
  u64 mine = 0;
  // offer one key a lane (0: none); every lane takes part
  __device__ __forceinline__ void offer(u64 key, int k) {
    const int lane = threadIdx.x & 31;
    u64 last = __shfl_sync(kFull, mine, k - 1);
    unsigned want = __ballot_sync(kFull, key > last);
    while (want) {
      const int src = __ffs(want) - 1;
      want &= want - 1;
      const u64 x = __shfl_sync(kFull, key, src);
      if (x <= last) continue;  // the last rose since the ballot
      const u64 up = __shfl_up_sync(kFull, mine, 1);
      const bool here = mine < x;                       // x goes at the first lane that holds less
      const bool before = lane > 0 && up < x;
      if (here) mine = before ? up : x;
      last = __shfl_sync(kFull, mine, k - 1);
    }
  }
};

// the k-th largest over the warp of one value a lane
__device__ __forceinline__ uint32_t kth_of_warp(uint32_t v, int k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {  // bitonic, falling
      const uint32_t w = __shfl_xor_sync(kFull, v, o);
      v = ((lane & size) == 0) == ((lane & o) == 0) ? max(v, w) : min(v, w);
    }
  return __shfl_sync(kFull, v, k - 1);
}

struct BeamSlice {
  double sum;  // of e^{logit - max}
  float max;
  float pad;
};

struct BeamK {
  ss_beam_args a;
  int slices, slice_len;  // slice_len: a multiple of the vector width
  int vec;
  BeamSlice* part;        // [batch * beams][slices]
  u64* keys;              // [batch * beams][slices][num_select]
};

template <typename IT>
__global__ void __launch_bounds__(kBsThreads) beam_slice_kernel(const __grid_constant__ BeamK P) {
  constexpr int VW = 16 / sizeof(IT);
  __shared__ float s_max[kBsWarps];
  __shared__ double s_sum[kBsWarps];
  __shared__ u64 s_keys[kBsWarps][32];
  griddep_launch_dependents();
  const ss_beam_args& a = P.a;
  const int row = blockIdx.x / P.slices, slice = blockIdx.x % P.slices;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, k = a.num_select;
  if (a.finished && a.finished[row]) return;  // the merge does not look at its slices
  const IT* x = static_cast<const IT*>(a.logits) + (int64_t)(row / a.beams) * a.logits_batch_stride +
                (int64_t)(row % a.beams) * a.logits_beam_stride;
  const int v0 = slice * P.slice_len, v1 = min(v0 + P.slice_len, a.vocab);
  WarpBest best;
  float m = -INFINITY, sum = 0.f;
  constexpr int E = 32, U = E / VW;  // values of a thread in a batch, 16-byte vectors of them under way at once
  for (int base = v0; base < v1; base += kBsThreads * E) {
    const int first = base + threadIdx.x * VW;  // vector u starts kBsThreads * VW * u further
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e0 = first + u * kBsThreads * VW;
      if (P.vec) {
        q[u] = ld_vector(x + e0, e0 + VW <= v1);
      }
      if (!P.vec || (e0 < v1 && e0 + VW > v1)) {
        union { uint4 v; IT e[VW]; } pk;
#pragma unroll
        for (int i = 0; i < VW; ++i) pk.e[i] = e0 + i < v1 ? x[e0 + i] : from_f<IT>(-INFINITY);
        q[u] = pk.v;
      }
    }
    const bool full = base + kBsThreads * E <= v1;  // the whole CTA's batch lies in the slice
    float vm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VW; ++i)  // what was read behind the slice's end is 0
        if (full || first + u * kBsThreads * VW + i < v1) vm = fmaxf(vm, to_f<IT>(reinterpret_cast<const IT*>(&q[u])[i]));
    if (vm > m) {
      sum *= expf(m - vm);  // 0 at the first finite value
      m = vm;
    }
    uint32_t bound = (uint32_t)(__shfl_sync(kFull, best.mine, k - 1) >> 32);
    if (base == v0) bound = kth_of_warp(first < v1 ? order_key(vm) : 0u, k);  // the list is empty
    const float floor_v = bound ? key_value(bound) : -INFINITY;
    const float mm = m == -INFINITY ? 0.f : m;
    uint32_t mask = 0;  // this lane's candidates
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const float v = to_f<IT>(reinterpret_cast<const IT*>(&q[u])[i]);
        if (full || first + u * kBsThreads * VW + i < v1) {
          (i & 1 ? s1 : s0) += expf(v - mm);  // an infinite maximum, or NaN, makes the sum NaN
          if (!(v < floor_v)) mask |= 1u << (u * VW + i);
        }
      }
    sum += s0 + s1;
    while (__any_sync(kFull, mask != 0)) {  // one of each lane at a time, read again
      u64 key = 0;
      if (mask) {
        const int e = __ffs(mask) - 1, at = first + e / VW * (kBsThreads * VW) + e % VW;
        mask &= mask - 1;
        key = ((u64)order_key(to_f<IT>(x[at])) << 32) | (uint32_t)~(uint32_t)at;
      }
      best.offer(key, k);
    }
  }
  // the CTA's maximum and sum
  float wm = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(kFull, wm, o));
  double ws = (m == -INFINITY && sum == 0.f) ? 0.0 : (double)sum * (double)expf(m - wm);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(kFull, ws, o);
  if (lane == 0) s_max[wid] = wm, s_sum[wid] = ws;
  s_keys[wid][lane] = lane < k ? best.mine : 0;
  __syncthreads();
  if (wid == 0) {
    float cm = -INFINITY;
    for (int i = 0; i < kBsWarps; ++i) cm = fmaxf(cm, s_max[i]);
    double cs = 0.0;
    for (int i = 0; i < kBsWarps; ++i)
      if (!(s_sum[i] == 0.0)) cs += s_sum[i] * (double)expf(s_max[i] - cm);
    for (int i = 1; i < kBsWarps; ++i) best.offer(s_keys[i][lane], k);
    const int64_t at = (int64_t)row * P.slices + slice;
    if (lane == 0) P.part[at] = BeamSlice{cs, cm, 0.f};
    if (lane < k) P.keys[at * k + lane] = best.mine;
  }
}

// order of the merge: larger value first, then the smaller flat index
__device__ __forceinline__ bool beats(double v, int i, double w, int j) { return v > w || (v == w && i < j); }

// the best 32 candidates of a warp, lane i the i-th best
struct WarpOrder {
  double v = -INFINITY;
  int i = INT32_MAX;
  // offer one candidate a lane (index INT32_MAX: none); every lane takes part
  __device__ __forceinline__ void offer(double x, int xi, int k) {
    const int lane = threadIdx.x & 31;
    double lv = __shfl_sync(kFull, v, k - 1);
    int li = __shfl_sync(kFull, i, k - 1);
    unsigned want = __ballot_sync(kFull, xi != INT32_MAX && beats(x, xi, lv, li));
    while (want) {
      const int src = __ffs(want) - 1;
      want &= want - 1;
      const double c = __shfl_sync(kFull, x, src);
      const int ci = __shfl_sync(kFull, xi, src);
      if (!beats(c, ci, lv, li)) continue;  // the last rose since the ballot
      const double uv = __shfl_up_sync(kFull, v, 1);
      const int ui = __shfl_up_sync(kFull, i, 1);
      const bool here = beats(c, ci, v, i);
      const bool before = lane > 0 && beats(c, ci, uv, ui);
      if (here) v = before ? uv : c, i = before ? ui : ci;
      lv = __shfl_sync(kFull, v, k - 1);
      li = __shfl_sync(kFull, i, k - 1);
    }
  }
};

// A beam's candidates from its logits again, in fp64: for a beam whose k-th best logit and a smaller one could give
// the same candidate, so that the order of the logits is not the order of the candidates.  `top` is the best of
// them: nothing behind k of those comes before them.  0.3 ms where all of 50280 tokens are read.
__device__ __forceinline__ WarpOrder beam_rescan(const ss_beam_args& a, int64_t at, double score, double lse, double top) {
  constexpr int U = 4;  // loads under way at a time
  WarpOrder best;
  for (int t0 = 0; t0 < a.vocab; t0 += 32 * U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + 32 * u + (threadIdx.x & 31);
      const int64_t e = at + min(t, a.vocab - 1);
      v[u] = a.io_dtype == SS_F32    ? static_cast<const float*>(a.logits)[e]
             : a.io_dtype == SS_BF16 ? to_f<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(a.logits)[e])
                                     : to_f<__half>(static_cast<const __half*>(a.logits)[e]);
    }
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
      const float x = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
      const int t = t0 + 32 * u + (threadIdx.x & 31);
      best.offer(score + ((double)x - lse), t < a.vocab ? t : INT32_MAX, a.num_select);
    }
    if (__shfl_sync(kFull, best.v, a.num_select - 1) == top) break;
  }
  return best;
}

// the next smaller float of a finite one
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x);
  return x == 0.f ? __uint_as_float(0x80000001u) : __uint_as_float(x > 0.f ? b - 1 : b + 1);
}

// One CTA per batch row, a warp per beam.
__global__ void __launch_bounds__(32 * SS_MAX_BEAMS) beam_merge_kernel(const __grid_constant__ BeamK P) {
  __shared__ double s_val[SS_MAX_BEAMS][32];
  __shared__ int s_tok[SS_MAX_BEAMS][32];
  const ss_beam_args& a = P.a;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, k = a.num_select;
  const int64_t row = (int64_t)blockIdx.x * a.beams + wid;
  const bool done = a.finished && a.finished[row];
  double score = a.scores[row];
  const bool dead = !(score < INFINITY);  // NaN or +infinity
  griddep_wait();
  double val = -INFINITY;
  int tok = -1;
  if (done) {
    // its score at the end token, then -infinity in the order of the tokens
    if (dead || score == -INFINITY) {
      tok = lane;
    } else if (lane == 0) {
      tok = a.eos_token;
      val = score;
    } else {
      tok = lane - 1 + (lane - 1 >= a.eos_token);
    }
  } else {
    float m = -INFINITY;
    const BeamSlice* part = P.part + row * P.slices;
    for (int s = lane; s < P.slices; s += 32) m = fmaxf(m, part[s].max);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    double sum = 0.0;
    for (int s = lane; s < P.slices; s += 32)
      if (!(part[s].sum == 0.0)) sum += part[s].sum * exp((double)part[s].max - (double)m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const double lse = (double)m + log(sum);
    WarpBest best;
    const u64* keys = P.keys + row * P.slices * k;
    const int n = P.slices * k;
    for (int i = 0; i < n; i += 32) best.offer(i + lane < n ? keys[i + lane] : 0, k);
    const float logit = key_value((uint32_t)(best.mine >> 32));
    const bool valid = lse > -INFINITY && lse < INFINITY && !dead && score > -INFINITY;  // false for NaN
    if (valid) {
      val = score + ((double)logit - lse);
      tok = best.mine ? (int)~(uint32_t)best.mine : -1;
      // candidates of -infinity follow in the order of the tokens, as the keys have them.  A finite logit next
      // below the last one's may give the same candidate (logits near zero, scores of a large magnitude)
      const bool same = lane == k - 1 && best.mine && logit > -INFINITY && val == score + ((double)below(logit) - lse);
      if (__any_sync(kFull, same)) {
        const int64_t at = (int64_t)blockIdx.x * a.logits_batch_stride + (int64_t)wid * a.logits_beam_stride;
        const WarpOrder order = beam_rescan(a, at, score, lse, __shfl_sync(kFull, val, 0));
        val = order.v;
        tok = order.i == INT32_MAX ? -1 : order.i;
      }
    } else {
      tok = lane;
    }
  }
  // a beam offers as many candidates as it has tokens
  if (lane >= k || lane >= a.vocab) tok = -1;
  s_val[wid][lane] = val;
  s_tok[wid][lane] = tok;
  __syncthreads();
  if (wid != 0) return;
  WarpOrder best;  // of the row
  for (int w = 0; w < a.beams; ++w) {
    const int t = s_tok[w][lane];
    best.offer(s_val[w][lane], t < 0 ? INT32_MAX : w * a.vocab + t, k);
  }
  if (lane < k) {
    const int64_t at = (int64_t)blockIdx.x * k + lane;
    a.out_scores[at] = (float)best.v;
    a.parents[at] = best.i / a.vocab;
    a.tokens[at] = best.i % a.vocab;
  }
}

// ------------------------------------------------------------------------------------ reordering
// Each thread owns one 16-byte (or 4-byte) column of a batch row's beams: it loads what its rows
// take from other beams, then stores, so the gather needs no second buffer.  Rows that keep their
// place are neither read nor written.  Bound by the memory traffic of the rows that move: 192 beams' states of
// 8 layers (179 MB, most of it moving) take 47 us.
struct ReorderK {
  ss_reorder_args a;
  int* status;
  int64_t first[SS_MAX_REORDER + 1];  // tensor i's first block of 256 columns
};

template <int W, typename V>
__device__ __forceinline__ void reorder_columns(char* rows, int64_t row_bytes, const int* from, int beams, int64_t col) {
  V v[W];
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < beams && from[w] != w) v[w] = *reinterpret_cast<const V*>(rows + from[w] * row_bytes + col);
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < beams && from[w] != w) *reinterpret_cast<V*>(rows + w * row_bytes + col) = v[w];
}

template <int W>
__global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ ReorderK P) {
  __shared__ int from[SS_MAX_BEAMS];
  const ss_reorder_args& a = P.a;
  griddep_wait();
  const int b = blockIdx.y;
  if (threadIdx.x < a.beams) {
    const int64_t p = a.parents[(int64_t)b * a.parents_batch_stride + threadIdx.x];
    const bool ok = p >= 0 && p < a.beams;
    from[threadIdx.x] = ok ? (int)p : threadIdx.x;
    if (!ok && blockIdx.x == 0 && P.status) atomicOr(P.status, kStatusParent);
  }
  __syncthreads();
  for (int64_t blk = blockIdx.x; blk < P.first[a.count]; blk += gridDim.x) {
    int i = 0;  // the block's tensor
    for (int hi = a.count; hi - i > 1;) {
      const int mid = (i + hi) / 2;
      if (P.first[mid] <= blk) i = mid;
      else hi = mid;
    }
    const int64_t bytes = a.row_bytes[i];
    char* rows = static_cast<char*>(a.data[i]) + (int64_t)b * a.beams * bytes;
    const bool wide = bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(a.data[i]) & 15) == 0;
    const int64_t at = (blk - P.first[i]) * 256 + threadIdx.x;
    if (wide) {
      if (at * 16 < bytes) reorder_columns<W, uint4>(rows, bytes, from, a.beams, at * 16);
    } else {
      if (at * 4 < bytes) reorder_columns<W, uint32_t>(rows, bytes, from, a.beams, at * 4);
    }
  }
}

}  // namespace ssb
