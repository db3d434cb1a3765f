// C ABI of the norms around a block (ss_block_norm_fwd / ss_block_norm_bwd): validation and dispatch
// over dtype, vectors a lane and warps a row.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/mamba_b200_ss.h"
#include "ss_block_norm.cuh"

namespace {

using namespace ssb;

// rows that start on a vector of 4 values
bool rows4(const void* p, int64_t stride, size_t es) {
  const uintptr_t m = 4 * es - 1;
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & m) == 0 && ((uintptr_t)(stride * (int64_t)es) & m) == 0);
}

bool weights16(const ss_block_norm_args& a) {
  return a.dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.post_weight) | reinterpret_cast<uintptr_t>(a.pre_weight) |
                             reinterpret_cast<uintptr_t>(a.scale)) & 15) == 0;
}

// the two roots of a row move as one 8-byte word
bool pairs(const float* rstd) { return (reinterpret_cast<uintptr_t>(rstd) & 7) == 0; }

struct Shape {
  int nv, wpr;  // vectors a lane, warps a row
};

// A row's warps: as few as hold it with 3 vectors of 4 values a lane, at most 8
Shape shape_of(int dim) {
  for (int wpr : {1, 2, 4, 8}) {
    const int need = (dim + 128 * wpr - 1) / (128 * wpr);
    if (need <= 3) return {need, wpr};
  }
  const int need = (dim + 1023) / 1024;
  return {need <= 4 ? 4 : need <= 6 ? 6 : 8, 8};
}

int sm_count() {
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaGetLastError();
  return sms;
}

// CTAs of the backward (the workspace holds two sums per column of each); the same rule wherever
// the library runs, so that ss_block_norm_work_elems needs no device
int bwd_ctas(int64_t rows, int wpr) {
  const int rpc = kBnWarps / wpr;
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + rpc - 1) / rpc, 2 * 148));
}

// rows that would overlap (the stride of a single row is not used)
bool short_rows(const ss_block_norm_args& a, int64_t stride) { return a.rows > 1 && stride < a.dim; }

int check(const ss_block_norm_args& a) {
  if (a.rows < 0 || a.dim < 1 || !(a.eps >= 0.f) || !(a.pre_eps >= 0.f) || !std::isfinite(a.scale_const)) return SS_ERR_INVALID;
  if (a.io_dtype != SS_F32 && a.io_dtype != SS_BF16 && a.io_dtype != SS_F16) return SS_ERR_UNSUPPORTED;
  if (a.activation < kActNone || a.activation > kActSigmoid) return SS_ERR_INVALID;
  if (a.dim > SS_MAX_BLOCK_NORM_DIM) return SS_ERR_UNSUPPORTED;
  if (a.rows == 0) return SS_OK;
  if (!a.y || !a.residual) return SS_ERR_INVALID;
  if (short_rows(a, a.y_row_stride) || short_rows(a, a.residual_row_stride)) return SS_ERR_INVALID;
  if (a.gate && a.gate_row_stride != 0 && short_rows(a, a.gate_row_stride)) return SS_ERR_INVALID;
  return SS_OK;
}

template <typename F>
int by_dtype(int io, F&& f) {
  switch (io) {
    case SS_F32: return record_cuda_status(f(float{}));
    case SS_BF16: return record_cuda_status(f(__nv_bfloat16{}));
    default: return record_cuda_status(f(__half{}));
  }
}

// the kernel's MODE of a call
int mode_of(const ss_block_norm_args& a, int vec, int wvec) {
  if (!vec || !wvec || !a.post_weight || !a.pre_weight) return kBnAny;
  if (!a.gate) return kBnPlain;
  return a.activation == kActSilu ? kBnGated : kBnAny;
}

template <typename IT, int NV, int WPR>
cudaError_t fwd(const BlockNormK& P, cudaStream_t st) {
  const int mode = mode_of(P.a, P.vec, P.wvec);
  auto kern = mode == kBnGated ? block_norm_fwd_kernel<IT, NV, WPR, kBnGated>
              : mode == kBnPlain ? block_norm_fwd_kernel<IT, NV, WPR, kBnPlain> : block_norm_fwd_kernel<IT, NV, WPR, kBnAny>;
  // as many CTAs as are resident at once, each walking its share of the rows: a second wave of a third of
  // them would take as long as the first
  static std::atomic<int> resident[3];
  int occ = resident[mode].load();
  if (occ == 0) {
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, 32 * kBnWarps, 0);
    if (e != cudaSuccess) return e;
    resident[mode].store(occ = std::max(occ, 1));
  }
  const int rpc = kBnWarps / WPR;
  const int64_t ctas = ((int64_t)P.a.rows + rpc - 1) / rpc;
  kern<<<(unsigned)std::min<int64_t>(ctas, (int64_t)occ * sm_count()), 32 * kBnWarps, 0, st>>>(P);
  return cudaGetLastError();
}

template <typename IT, int NV, int WPR>
cudaError_t bwd(const BlockNormBwdK& P, cudaStream_t st) {
  const int mode = P.a.dh ? mode_of(P.a.f, P.vec, P.wvec) : kBnAny;
  auto kern = mode == kBnGated ? block_norm_bwd_kernel<IT, NV, WPR, kBnGated>
              : mode == kBnPlain ? block_norm_bwd_kernel<IT, NV, WPR, kBnPlain> : block_norm_bwd_kernel<IT, NV, WPR, kBnAny>;
  const size_t smem = sizeof(float) * NV * WPR * 32 * kBv +  // column sums; the next row's vectors
                      (mode == kBnAny ? 0 : (sizeof(IT) == 2 ? 2 : 1) * (mode == kBnGated ? 5 : 4) * NV * sizeof(typename BnVec<IT>::T) * 32 * kBnWarps);
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), smem + 256);  // and the static part
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)bwd_ctas(P.a.f.rows, WPR), 32 * kBnWarps, smem, st>>>(P);
  return cudaGetLastError();
}

}  // namespace

// a row that did not fit half as many warps has at least 2 vectors a lane
#define SSB_BN_SHAPES(F)                                            \
  if (s.wpr == 1) {                                                 \
    if (s.nv == 1) return F<IT, 1, 1>(P, st);                       \
    return s.nv == 2 ? F<IT, 2, 1>(P, st) : F<IT, 3, 1>(P, st);     \
  }                                                                 \
  if (s.wpr == 2) return s.nv <= 2 ? F<IT, 2, 2>(P, st) : F<IT, 3, 2>(P, st); \
  if (s.wpr == 4) return s.nv <= 2 ? F<IT, 2, 4>(P, st) : F<IT, 3, 4>(P, st); \
  if (s.nv <= 2) return F<IT, 2, 8>(P, st);                         \
  if (s.nv <= 3) return F<IT, 3, 8>(P, st);                         \
  if (s.nv <= 4) return F<IT, 4, 8>(P, st);                         \
  if (s.nv <= 6) return F<IT, 6, 8>(P, st);                         \
  return F<IT, 8, 8>(P, st);

extern "C" {

size_t ss_block_norm_work_elems(int64_t rows, int dim, int io_dtype) {
  (void)io_dtype;
  if (rows < 1 || dim < 1 || dim > SS_MAX_BLOCK_NORM_DIM) return 0;
  return (size_t)bwd_ctas(rows, shape_of(dim).wpr) * 2 * dim;
}

int ss_block_norm_fwd(const ss_block_norm_args* a, void* stream) {
  if (a == nullptr) return SS_ERR_INVALID;
  const int rc = check(*a);
  if (rc != SS_OK) return rc;
  if (a->rows == 0) return SS_OK;
  if (!a->h || short_rows(*a, a->h_row_stride) || !pairs(a->rstd)) return SS_ERR_INVALID;
  if (a->pre_weight && (!a->x || short_rows(*a, a->x_row_stride))) return SS_ERR_INVALID;
  const size_t es = a->io_dtype == SS_F32 ? 4 : 2;
  BlockNormK P;
  P.a = *a;
  P.wvec = weights16(*a);
  P.vec = a->dim % 4 == 0 && rows4(a->y, a->y_row_stride, es) &&
          rows4(a->residual, a->residual_row_stride, es) && rows4(a->gate, a->gate_row_stride, es) &&
          rows4(a->h, a->h_row_stride, es) && (!a->pre_weight || rows4(a->x, a->x_row_stride, es));
  cudaStream_t st = (cudaStream_t)stream;
  return by_dtype(a->io_dtype, [&](auto tag) -> cudaError_t {
    using IT = decltype(tag);
    const Shape s = shape_of(a->dim);
    SSB_BN_SHAPES(fwd)
  });
}

int ss_block_norm_bwd(const ss_block_norm_bwd_args* g, void* stream) {
  if (g == nullptr) return SS_ERR_INVALID;
  const ss_block_norm_args& a = g->f;
  const int rc = check(a);
  if (rc != SS_OK) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const float ofs = a.unit_offset ? 1.f : 0.f;
  const size_t es = a.io_dtype == SS_F32 ? 4 : 2;
  const Shape s = shape_of(a.dim);
  if (a.rows > 0) {
    if (!a.rstd || !pairs(a.rstd) || !g->dresidual || !g->dy || !g->work || (a.gate && !g->dgate) || (a.pre_weight && !g->dx))
      return SS_ERR_INVALID;
    if (short_rows(a, g->dy_row_stride) || short_rows(a, g->dresidual_row_stride) ||
        (a.gate && short_rows(a, g->dgate_row_stride)) || (a.pre_weight && short_rows(a, g->dx_row_stride)) ||
        (g->dh && short_rows(a, g->dh_row_stride)))
      return SS_ERR_INVALID;
    BlockNormBwdK P;
    P.a = *g;
    P.wvec = weights16(a);
    P.vec = a.dim % 4 == 0 && rows4(a.y, a.y_row_stride, es) &&
            rows4(a.residual, a.residual_row_stride, es) && rows4(a.gate, a.gate_row_stride, es) &&
            (!a.pre_weight || rows4(g->dx, g->dx_row_stride, es)) && rows4(g->dh, g->dh_row_stride, es) &&
            rows4(g->dy, g->dy_row_stride, es) && rows4(g->dresidual, g->dresidual_row_stride, es) &&
            (!a.gate || rows4(g->dgate, g->dgate_row_stride, es));
    const int r = by_dtype(a.io_dtype, [&](auto tag) -> cudaError_t {
      using IT = decltype(tag);
      SSB_BN_SHAPES(bwd)
    });
    if (r != SS_OK) return r;
  }
  if (!g->dpost_weight && !g->dpre_weight && !g->dscale) return SS_OK;
  const dim3 grid((unsigned)((a.dim + 31) / 32), 2);
  block_norm_cols_kernel<<<grid, 1024, 0, st>>>(g->work, a.rows > 0 ? bwd_ctas(a.rows, s.wpr) : 0, a.dim, a.post_weight,
                                               a.scale, a.scale_const, ofs, g->dpost_weight, g->dpre_weight, g->dscale);
  return record_cuda_status(cudaGetLastError());
}

}  // extern "C"
