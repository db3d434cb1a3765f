// C ABI of linear attention: validation, the runs of the recurrence that make up a call, the
// segments that a long sequence is cut into, and dispatch.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/mamba_b200_ss.h"
#include "ss_linear.cuh"
#include "ss_linear_tc.cuh"

namespace {

using namespace ssb;

int sm_count() {
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaGetLastError();
  return sms;
}

size_t align16(size_t n) { return (n + 15) & ~size_t(15); }

int tiles_of(int dim) { return (dim + kLsN - 1) / kLsN; }

bool sizes_ok(const ss_linear_args& a) {
  return a.batch >= 0 && a.seqlen >= 0 && a.heads >= 1 && a.key_heads >= 1 && a.heads % a.key_heads == 0 &&
         a.key_dim >= 1 && a.value_dim >= 1;
}

// what the kernels' indexes hold
bool limits_ok(const ss_linear_args& a) {
  return a.key_dim <= SS_MAX_LINEAR_DIM && a.value_dim <= SS_MAX_LINEAR_DIM && (int64_t)a.batch * a.heads <= (1 << 24) &&
         a.seqlen <= (1 << 30);
}

bool dtypes_ok(int io, int decay) {
  return (io == SS_F32 || io == SS_BF16 || io == SS_F16) && (decay == SS_F32 || decay == io);
}

// Segments that run side by side: enough CTAs for the GPU (`slots`) when batch x heads are few, at least two
// chunks each, at most 32.  A segment's own state costs half to four fifths of what its outputs cost, and the
// first segment neither needs nor waits for the states of the others.  Where two CTAs share an SM (narrow fp32
// heads) it starts beside their first pass (a programmatic launch) and is half as long again: 8 x 1024 tokens of
// 12 heads of 64 take 151 us, 161 in equal segments.  Where a CTA fills its SM there is no room beside it, and
// the segments are equal: 1 x 16384 tokens of 16 heads of 128 x 128 in bf16 take 151 us, 179 with a longer first.
struct Split {
  int segs, first, chunks;
};

Split split_of(const ss_linear_args& a, int chunk, int passes, int tiles, bool two) {
  const int n = (a.seqlen + chunk - 1) / chunk;
  const int64_t ctas = (int64_t)a.batch * a.heads * passes * tiles;
  const int slots = two ? 2 * 148 : 148;
  int segs = 1;
  if (ctas > 0 && ctas < slots) segs = (int)std::max<int64_t>(1, std::min<int64_t>({slots / ctas, n / 2, 32}));
  Split s{1, std::max(n, 1), std::max(n, 1)};
  if (segs > 1) {
    s.chunks = two ? std::max(1, (2 * n + 2 * segs) / (2 * segs + 1)) : (n + segs - 1) / segs;  // n / (segs + 1/2)
    s.first = std::min(n - 1, std::max(s.chunks, n - (segs - 1) * s.chunks));
    s.segs = 1 + (n - s.first + s.chunks - 1) / s.chunks;
  }
  return s;
}

// The scratch of a call, cut into its parts (offsets in bytes; absent parts are -1).  The segments of
// both kernels fit.
struct Work {
  size_t bytes = 0;
  int64_t sums = -1, seg_decay = -1, dots = -1, parts = -1;
  Split simt, tc;
};

size_t dot_bytes(int io) { return io == SS_F32 ? sizeof(LinDot<float>) : sizeof(LinDot<__half>); }

Work work_of(const ss_linear_args& a, int backward) {
  Work w;
  const int passes = backward ? 3 : 1;
  const int tiles = backward ? std::max(tiles_of(a.key_dim), tiles_of(a.value_dim)) : tiles_of(a.value_dim);
  w.simt = split_of(a, kLsC, passes, tiles, std::max(a.key_dim, a.value_dim) <= kLsN);
  w.tc = a.io_dtype == SS_F32 ? Split{1, 1, 1} : split_of(a, kTcC, passes, tiles, false);
  const int segs = a.io_dtype == SS_F32 ? w.simt.segs : std::max(w.simt.segs, w.tc.segs);
  const size_t bh = (size_t)a.batch * a.heads;
  auto take = [&](size_t n) {
    const int64_t at = (int64_t)w.bytes;
    w.bytes += align16(n);
    return at;
  };
  if (segs > 1) {
    w.sums = take(sizeof(float) * passes * bh * segs * a.key_dim * a.value_dim);
    w.seg_decay = take(sizeof(float) * 2 * bh * segs);
  }
  if (backward) {
    w.dots = take(dot_bytes(a.io_dtype) * 2 * tiles_of(a.key_dim) * bh * a.seqlen);
    if (a.heads != a.key_heads) w.parts = take(sizeof(float) * 2 * bh * a.seqlen * a.key_dim);
  }
  return w;
}

// a launch that may start before the kernel ahead of it in the stream has ended (it waits where it has to)
template <typename K>
cudaError_t launch_early(void (*kern)(K), dim3 grid, int threads, size_t smem, const K& P, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P);
}

cudaError_t launch_fold(const LinK& P, int passes, cudaStream_t st) {
  int64_t block = 0;
  for (int i = 0; i < passes; ++i) block = std::max<int64_t>(block, (int64_t)P.pass[i].dk * P.pass[i].dv);
  const dim3 grid((unsigned)((block + 255) / 256), (unsigned)(P.batch * P.heads), (unsigned)passes);
  return launch_early(linear_fold_kernel, grid, 256, 0, P, st);
}

template <typename IT, int DMAX>
cudaError_t run_simt(const LinK& P, int passes, cudaStream_t st) {
  constexpr size_t smem = sizeof(LsSmem<DMAX>);
  auto main_k = linear_simt_kernel<IT, DMAX, false>;
  auto sum_k = linear_simt_kernel<IT, DMAX, true>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(main_k), smem);
  if (e == cudaSuccess) e = ensure_smem_limit(reinterpret_cast<const void*>(sum_k), smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((int64_t)P.batch * P.heads * P.segs), (unsigned)(passes * (DMAX / kLsN)));
  if (P.segs > 1) {
    sum_k<<<grid, kLsThreads, smem, st>>>(P);
    e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_fold(P, passes, st);
    if (e != cudaSuccess) return e;
    return launch_early(main_k, grid, kLsThreads, smem, P, st);
  }
  main_k<<<grid, kLsThreads, smem, st>>>(P);
  return cudaGetLastError();
}

// one launch over passes [pass0, pass0 + n) of T
template <typename IT, int MODE>
cudaError_t launch_tc(LinTcK& T, int pass0, int n, bool early, cudaStream_t st) {
  constexpr size_t most = std::max(TcShape<64>::kBytes, TcShape<128>::kBytes);
  static_assert(most <= 232448, "shared memory of a CTA");
  static_assert(sizeof(TcBars) <= kBarBytes, "barriers");
  auto kern = linear_tc_kernel<IT, MODE>;
  const cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), most);
  if (e != cudaSuccess) return e;
  T.pass0 = pass0;
  T.tiles = 1;
  bool wide = false;
  for (int i = pass0; i < pass0 + n; ++i) {
    T.tiles = std::max(T.tiles, (T.k.pass[i].dv + kTcN - 1) / kTcN);
    wide |= T.k.pass[i].dk > 64;
  }
  T.parts = n * T.tiles;
  const dim3 grid((unsigned)((int64_t)T.k.batch * T.k.heads * T.k.segs * T.parts));
  const size_t smem = wide ? most : (size_t)TcShape<64>::kBytes;
  if (early) return launch_early(kern, grid, kTcThreads, smem, T, st);
  kern<<<grid, kTcThreads, smem, st>>>(T);
  return cudaGetLastError();
}

// The passes' segments and fold, then the gradients with dot products (the first `grads`), then the others.
// Every launch but the first may start while the one ahead of it ends: its first segments need nothing of it.
template <typename IT>
cudaError_t launch_all(LinTcK& T, int passes, int grads, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  bool early = false;
  if (T.k.segs > 1) {
    e = launch_tc<IT, kTcState>(T, 0, passes, false, st);
    if (e == cudaSuccess) e = launch_fold(T.k, passes, st);
    early = true;
  }
  if (e == cudaSuccess && grads > 0) {
    e = launch_tc<IT, kTcGrad>(T, 0, grads, early, st);
    early = true;
  }
  if (e == cudaSuccess && grads < passes) {
    bool state = false;  // fp16 keeps 22 bits in two parts and needs no other kernel
    for (int i = grads; i < passes; ++i) state |= T.k.pass[i].s_out != nullptr && std::is_same<IT, __nv_bfloat16>::value;
    if constexpr (std::is_same<IT, __nv_bfloat16>::value) {
      if (state) return launch_tc<IT, kTcOutState>(T, grads, passes - grads, early, st);
    }
    e = launch_tc<IT, kTcOut>(T, grads, passes - grads, early, st);
  }
  return e;
}

// rows of whole 16-byte units; the stride of an axis of one element is never stepped along, here as in map_heads
bool vec16(const LinK& P, const void* p, int heads, int es, int64_t b, int64_t l, int64_t h) {
  auto whole = [&](int n, int64_t stride) { return n <= 1 || ((stride * es) & 15) == 0; };
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && whole(P.batch, b) && whole(P.seqlen, l) && whole(heads, h);
}

// The tensor-core kernel takes every 16-bit call whose rows are whole 16-byte units (TMA loads, vector
// stores); false: it cannot.
bool run_tc(int io, const LinK& P, int passes, cudaStream_t st, cudaError_t* e) {
  LinTcK T;
  int grads = 0;
  for (int i = 0; i < passes; ++i) {
    const LinPass& A = P.pass[i];
    if (A.dk % 8 || A.dv % 8 || !vec16(P, A.o, P.heads, A.o_f32 ? 4 : 2, A.ob, A.ol, A.oh) ||
        (A.dot && !vec16(P, A.p, P.heads / A.rp, 2, A.pb, A.pl, A.ph)))
      return false;
    const struct {
      const void* p;
      int64_t d, b, l, h;
      int r;
    } x[3] = {{A.q, A.dk, A.qb, A.ql, A.qh, A.rq}, {A.k, A.dk, A.kb, A.kl, A.kh, A.rk}, {A.v, A.dv, A.vb, A.vl, A.vh, A.rv}};
    for (int j = 0; j < 4; ++j) {
      const bool ok = j < 3 ? map_heads(&T.map[i][j], x[j].p, io, x[j].d, P.heads / x[j].r, P.seqlen, P.batch, x[j].h, x[j].l,
                                        x[j].b, kTcC)
                            : map_heads(&T.map[i][3], A.o, A.o_f32 ? SS_F32 : io, A.dv, P.heads, P.seqlen, P.batch, A.oh,
                                        A.ol, A.ob, 32);
      if (!ok) return false;
    }
    grads += A.dot || A.o_f32;  // they come first
  }
  T.k = P;
  T.status = device_status_word();
  T.wait_limit = wait_limit();
  *e = io == SS_BF16 ? launch_all<__nv_bfloat16>(T, passes, grads, st) : launch_all<__half>(T, passes, grads, st);
  return true;
}

cudaError_t run_passes(int io, LinK& P, const Work& w, int passes, cudaStream_t st) {
  if (io != SS_F32 && P.seqlen > 0) {
    P.segs = w.tc.segs, P.seg_first = w.tc.first, P.seg_chunks = w.tc.chunks;
    cudaError_t e;
    if (run_tc(io, P, passes, st, &e)) return e;
  }
  P.segs = w.simt.segs, P.seg_first = w.simt.first, P.seg_chunks = w.simt.chunks;
  bool wide = false;
  for (int i = 0; i < passes; ++i) wide |= P.pass[i].dk > 64 || P.pass[i].dv > 64;
  switch (io) {
    case SS_F32: return wide ? run_simt<float, 128>(P, passes, st) : run_simt<float, 64>(P, passes, st);
    case SS_BF16: return run_simt<__nv_bfloat16, 128>(P, passes, st);
    default: return run_simt<__half, 128>(P, passes, st);
  }
}

LinK problem(const ss_linear_args& a, const Work& w, void* work) {
  LinK P{};
  P.g = a.log_decay;
  P.g_f32 = a.decay_dtype == SS_F32;
  P.gb = a.decay_batch_stride, P.gl = a.decay_seq_stride, P.gh = a.decay_head_stride;
  P.lens = a.seq_lens;
  P.batch = a.batch, P.seqlen = a.seqlen, P.heads = a.heads;
  if (w.seg_decay >= 0) P.seg_decay = reinterpret_cast<float*>(static_cast<char*>(work) + w.seg_decay);
  return P;
}

bool work_ok(const Work& w, const void* p) { return !w.bytes || (p && (reinterpret_cast<uintptr_t>(p) & 15) == 0); }

// status of the arguments that both directions share (a zero batch may carry null pointers)
int check_fwd(const ss_linear_args& a) {
  if (!sizes_ok(a)) return SS_ERR_INVALID;
  if (!dtypes_ok(a.io_dtype, a.decay_dtype)) return SS_ERR_UNSUPPORTED;
  if (!limits_ok(a)) return SS_ERR_UNSUPPORTED;
  if (!std::isnormal(a.scale)) return SS_ERR_INVALID;  // its reciprocal is needed too
  const bool empty = a.batch == 0 || a.seqlen == 0;
  if (!empty && (!a.q || !a.k || !a.v || !a.log_decay)) return SS_ERR_INVALID;
  return SS_OK;
}

}  // namespace

extern "C" {

size_t ss_linear_work_bytes(const ss_linear_args* a, int backward) {
  if (a == nullptr || !sizes_ok(*a) || !limits_ok(*a)) return 0;
  return work_of(*a, backward != 0).bytes;
}

int ss_linear_fwd(const ss_linear_args* a, void* stream) {
  if (a == nullptr) return SS_ERR_INVALID;
  const int rc = check_fwd(*a);
  if (rc != SS_OK) return rc;
  if (a->batch == 0) return SS_OK;
  if (a->seqlen > 0 && !a->o) return SS_ERR_INVALID;
  if (a->seqlen == 0 && !a->state_out) return SS_OK;
  const Work w = work_of(*a, 0);
  if (!work_ok(w, a->work)) return SS_ERR_INVALID;
  LinK P = problem(*a, w, a->work);
  LinPass& A = P.pass[0];
  const int rep = a->heads / a->key_heads;
  A.q = a->q, A.qb = a->q_batch_stride, A.ql = a->q_seq_stride, A.qh = a->q_head_stride, A.rq = rep;
  A.k = a->k, A.kb = a->k_batch_stride, A.kl = a->k_seq_stride, A.kh = a->k_head_stride, A.rk = rep;
  A.v = a->v, A.vb = a->v_batch_stride, A.vl = a->v_seq_stride, A.vh = a->v_head_stride, A.rv = 1;
  A.o = a->o, A.ob = a->o_batch_stride, A.ol = a->o_seq_stride, A.oh = a->o_head_stride;
  A.dk = a->key_dim, A.dv = a->value_dim;
  A.scale = a->scale;
  A.s_in = a->state_in, A.s_in_scale = 1.f;
  A.s_out = a->state_out, A.s_out_scale = 1.f;
  A.s_row = a->value_dim, A.s_col = 1;
  if (w.sums >= 0) A.sum = reinterpret_cast<float*>(static_cast<char*>(a->work) + w.sums);
  return record_cuda_status(run_passes(a->io_dtype, P, w, 1, (cudaStream_t)stream));
}

int ss_linear_bwd(const ss_linear_bwd_args* g, void* stream) {
  if (g == nullptr) return SS_ERR_INVALID;
  const ss_linear_args& a = g->f;
  const int rc = check_fwd(a);
  if (rc != SS_OK) return rc;
  if (a.batch == 0) {  // the one result that no rows leave something of: a decay per head, whose gradient is zero
    if (!g->dlog_decay || a.decay_batch_stride || a.decay_seq_stride) return SS_OK;
    const size_t es = a.decay_dtype == SS_F32 ? 4 : 2;
    return record_cuda_status(cudaMemsetAsync(g->dlog_decay, 0, es * a.heads, (cudaStream_t)stream));
  }
  if (a.seqlen > 0 && (!g->dout || !g->dq || !g->dk || !g->dv)) return SS_ERR_INVALID;
  if (g->dstate_out && g->dlog_decay && !a.state_out) return SS_ERR_INVALID;
  const Work w = work_of(a, 1);
  if (!work_ok(w, g->work)) return SS_ERR_INVALID;
  char* base = static_cast<char*>(g->work);
  LinK P = problem(a, w, base);
  const int rep = a.heads / a.key_heads;
  const int64_t bh = (int64_t)a.batch * a.heads, block = (int64_t)a.key_dim * a.value_dim;
  const int tq = tiles_of(a.key_dim);
  char* dots = g->dlog_decay ? base + w.dots : nullptr;
  const int64_t dots_of_one = (int64_t)dot_bytes(a.io_dtype) * tq * bh * a.seqlen;
  float* parts = w.parts >= 0 ? reinterpret_cast<float*>(base + w.parts) : nullptr;
  float* sums = w.sums >= 0 ? reinterpret_cast<float*>(base + w.sums) : nullptr;
  struct T {
    const void* p;
    int64_t b, l, h;
    int rep;
  };
  const T q{a.q, a.q_batch_stride, a.q_seq_stride, a.q_head_stride, rep};
  const T k{a.k, a.k_batch_stride, a.k_seq_stride, a.k_head_stride, rep};
  const T v{a.v, a.v_batch_stride, a.v_seq_stride, a.v_head_stride, 1};
  const T dout{g->dout, g->do_batch_stride, g->do_seq_stride, g->do_head_stride, 1};
  auto set = [&](int i, const T& x, const T& y, const T& z, int dk, int dv, bool reverse) -> LinPass& {
    LinPass& A = P.pass[i];
    A.q = x.p, A.qb = x.b, A.ql = x.l, A.qh = x.h, A.rq = x.rep;
    A.k = y.p, A.kb = y.b, A.kl = y.l, A.kh = y.h, A.rk = y.rep;
    A.v = z.p, A.vb = z.b, A.vl = z.l, A.vh = z.h, A.rv = z.rep;
    A.dk = dk, A.dv = dv, A.reverse = reverse, A.scale = a.scale;
    A.s_in_scale = reverse ? 1.f / a.scale : 1.f;  // a reverse run's state times scale is the state's gradient
    if (sums) A.sum = sums + (int64_t)i * bh * std::max(w.simt.segs, w.tc.segs) * block;
    return A;
  };
  auto grad = [&](LinPass& A, int i, void* out, int64_t b, int64_t l, int64_t h, const T& p) {
    if (parts) {  // fp32 parts per head, summed below
      A.o = parts + (int64_t)i * bh * a.seqlen * a.key_dim;
      A.o_f32 = 1;
      A.oh = a.key_dim, A.ol = (int64_t)a.heads * a.key_dim, A.ob = (int64_t)a.seqlen * A.ol;
    } else {
      A.o = out, A.ob = b, A.ol = l, A.oh = h;
    }
    if (dots) {
      A.dot = reinterpret_cast<float*>(dots + i * dots_of_one);
      A.p = p.p, A.pb = p.b, A.pl = p.l, A.ph = p.h, A.rp = p.rep;
    }
  };
  LinPass& Q = set(0, dout, v, k, a.value_dim, a.key_dim, false);
  grad(Q, 0, g->dq, g->dq_batch_stride, g->dq_seq_stride, g->dq_head_stride, q);
  Q.s_in = a.state_in, Q.s_row = 1, Q.s_col = a.value_dim;
  LinPass& K = set(1, v, dout, q, a.value_dim, a.key_dim, true);
  grad(K, 1, g->dk, g->dk_batch_stride, g->dk_seq_stride, g->dk_head_stride, k);
  K.s_in = g->dstate_out, K.s_row = 1, K.s_col = a.value_dim;
  LinPass& V = set(2, k, q, dout, a.key_dim, a.value_dim, true);
  V.o = g->dv, V.ob = g->dv_batch_stride, V.ol = g->dv_seq_stride, V.oh = g->dv_head_stride;
  V.s_in = g->dstate_out, V.s_row = a.value_dim, V.s_col = 1;
  V.s_out = g->dstate_in, V.s_out_scale = a.scale;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = run_passes(a.io_dtype, P, w, 3, st);
  if (e != cudaSuccess) return record_cuda_status(e);
  if (parts && a.seqlen > 0) {
    LinGroupK G{};
    G.batch = a.batch, G.seqlen = a.seqlen, G.key_heads = a.key_heads, G.rep = rep, G.dim = a.key_dim;
    G.parts[0] = parts, G.out[0] = g->dq, G.ob[0] = g->dq_batch_stride, G.ol[0] = g->dq_seq_stride, G.oh[0] = g->dq_head_stride;
    G.parts[1] = parts + bh * a.seqlen * a.key_dim;
    G.out[1] = g->dk, G.ob[1] = g->dk_batch_stride, G.ol[1] = g->dk_seq_stride, G.oh[1] = g->dk_head_stride;
    const bool v4 = a.key_dim % 4 == 0;  // the parts start on 16 bytes then
    const int64_t n = (int64_t)a.batch * a.seqlen * a.key_heads * (v4 ? a.key_dim / 4 : a.key_dim);
    const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 8 * sm_count()), 2);
    auto sum = [&](auto tag) {
      using IT = decltype(tag);
      if (v4) linear_group_sum_kernel<IT, 4><<<grid, 256, 0, st>>>(G);
      else linear_group_sum_kernel<IT, 1><<<grid, 256, 0, st>>>(G);
    };
    if (a.io_dtype == SS_F32) sum(float{});
    else if (a.io_dtype == SS_BF16) sum(__nv_bfloat16{});
    else sum(__half{});
    e = cudaGetLastError();
    if (e != cudaSuccess) return record_cuda_status(e);
  }
  if (g->dlog_decay) {
    LinDecayK D{};
    D.xq = dots, D.yk = dots + dots_of_one, D.tq = D.tk = tq;
    if (g->dstate_out) D.d_last = g->dstate_out, D.last = a.state_out;
    D.block = block;
    D.g = a.log_decay, D.dg = g->dlog_decay;
    D.g_f32 = a.decay_dtype == SS_F32, D.g_bf16 = a.io_dtype == SS_BF16;
    D.per_head = a.decay_batch_stride == 0 && a.decay_seq_stride == 0;
    D.gb = a.decay_batch_stride, D.gl = a.decay_seq_stride, D.gh = a.decay_head_stride;
    D.lens = a.seq_lens;
    D.batch = a.batch, D.seqlen = a.seqlen, D.heads = a.heads;
    const unsigned ctas = (unsigned)(D.per_head ? a.heads : bh);
    if (a.io_dtype == SS_F32) linear_decay_grad_kernel<LinDot<float>><<<ctas, kLdThreads, 0, st>>>(D);
    else linear_decay_grad_kernel<LinDot<__half>><<<ctas, kLdThreads, 0, st>>>(D);
    e = cudaGetLastError();
  }
  return record_cuda_status(e);
}

int ss_linear_step(const ss_linear_step_args* a, void* stream) {
  if (a == nullptr) return SS_ERR_INVALID;
  if (a->batch < 0 || a->heads < 1 || a->key_heads < 1 || a->heads % a->key_heads != 0 || a->key_dim < 1 ||
      a->value_dim < 1 || !std::isfinite(a->scale))
    return SS_ERR_INVALID;
  if (!dtypes_ok(a->io_dtype, a->decay_dtype)) return SS_ERR_UNSUPPORTED;
  if (a->key_dim > SS_MAX_LINEAR_DIM || a->value_dim > SS_MAX_LINEAR_DIM) return SS_ERR_UNSUPPORTED;
  if ((int64_t)a->batch * a->heads > 2147483647LL) return SS_ERR_UNSUPPORTED;
  if (a->batch == 0) return SS_OK;
  if (!a->state || !a->q || !a->k || !a->v || !a->log_decay || !a->o) return SS_ERR_INVALID;
  if (a->state_batch_stride < (int64_t)a->heads * a->key_dim * a->value_dim) return SS_ERR_INVALID;
  LinStepK P;
  P.a = *a;
  P.vec = a->value_dim % 4 == 0 && a->state_batch_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a->state) & 15) == 0;
  const unsigned grid = (unsigned)((int64_t)a->batch * a->heads);
  cudaStream_t st = (cudaStream_t)stream;
  auto step = [&](auto tag) {
    using IT = decltype(tag);
    if (a->value_dim <= 32) linear_step_kernel<IT, 8><<<grid, 32 * kLstWarps, 0, st>>>(P);
    else if (a->value_dim <= 64) linear_step_kernel<IT, 16><<<grid, 32 * kLstWarps, 0, st>>>(P);
    else linear_step_kernel<IT, 32><<<grid, 32 * kLstWarps, 0, st>>>(P);
  };
  if (a->io_dtype == SS_F32) step(float{});
  else if (a->io_dtype == SS_BF16) step(__nv_bfloat16{});
  else step(__half{});
  return record_cuda_status(cudaGetLastError());
}

}  // extern "C"
