// C ABI of the beam-search step (ss_beam_select, ss_reorder): validation, slices and dispatch.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mamba_b200_ss.h"
#include "ss_beam.cuh"

namespace {

using namespace ssb;

// slices of a beam's vocabulary: about three CTAs per SM over all beams (a longer slice offers fewer of its
// logits: 192 beams x 50280 fp32 take 55 us in slices of 8 thousand, 51 us in these, both kernels), at least 1024
// tokens each
int slices_of(int64_t rows, int vocab) {
  const int64_t want = std::max<int64_t>(1, (3 * 148 + rows - 1) / std::max<int64_t>(1, rows));
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (vocab + 2047) / 2048, 64}));
}

bool sizes_ok(int batch, int beams, int vocab, int k) {
  return batch >= 0 && beams >= 1 && vocab >= 1 && k >= 1 && (int64_t)k <= (int64_t)beams * vocab;
}

bool limits_ok(int beams, int vocab, int k) {
  return beams <= SS_MAX_BEAMS && k <= 32 && (int64_t)beams * vocab <= (1 << 30);
}

template <typename K>
cudaError_t launch_dependent(void (*kern)(K), dim3 grid, int threads, const K& P, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P);
}

}  // namespace

extern "C" {

size_t ss_beam_work_bytes(int batch, int beams, int vocab, int num_select) {
  if (!sizes_ok(batch, beams, vocab, num_select) || !limits_ok(beams, vocab, num_select) || batch == 0) return 0;
  const int64_t rows = (int64_t)batch * beams;
  return (size_t)rows * slices_of(rows, vocab) * (sizeof(BeamSlice) + sizeof(u64) * num_select);
}

int ss_beam_select(const ss_beam_args* a, void* stream) {
  if (a == nullptr) return SS_ERR_INVALID;
  if (!sizes_ok(a->batch, a->beams, a->vocab, a->num_select)) return SS_ERR_INVALID;
  if (a->io_dtype != SS_F32 && a->io_dtype != SS_BF16 && a->io_dtype != SS_F16) return SS_ERR_UNSUPPORTED;
  if (!limits_ok(a->beams, a->vocab, a->num_select)) return SS_ERR_UNSUPPORTED;
  if (a->finished && (a->eos_token < 0 || a->eos_token >= a->vocab)) return SS_ERR_INVALID;
  if (a->batch == 0) return SS_OK;
  if (!a->logits || !a->scores || !a->out_scores || !a->parents || !a->tokens || !a->work ||
      (reinterpret_cast<uintptr_t>(a->work) & 15))
    return SS_ERR_INVALID;
  if (a->logits_batch_stride < 0 || a->logits_beam_stride < 0) return SS_ERR_INVALID;
  const int64_t rows = (int64_t)a->batch * a->beams;
  const size_t es = a->io_dtype == SS_F32 ? 4 : 2;
  const int vw = (int)(16 / es);
  BeamK P;
  P.a = *a;
  P.slices = slices_of(rows, a->vocab);
  P.slice_len = ((a->vocab + P.slices - 1) / P.slices + vw - 1) / vw * vw;
  P.vec = (reinterpret_cast<uintptr_t>(a->logits) & 15) == 0 && (a->logits_batch_stride * (int64_t)es) % 16 == 0 &&
          (a->logits_beam_stride * (int64_t)es) % 16 == 0;
  P.part = static_cast<BeamSlice*>(a->work);
  P.keys = reinterpret_cast<u64*>(P.part + rows * P.slices);
  if (rows * P.slices > 2147483647LL) return SS_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(rows * P.slices);
  switch (a->io_dtype) {
    case SS_F32: beam_slice_kernel<float><<<grid, kBsThreads, 0, st>>>(P); break;
    case SS_BF16: beam_slice_kernel<__nv_bfloat16><<<grid, kBsThreads, 0, st>>>(P); break;
    default: beam_slice_kernel<__half><<<grid, kBsThreads, 0, st>>>(P); break;
  }
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_dependent(beam_merge_kernel, dim3((unsigned)a->batch), 32 * a->beams, P, st);
  return record_cuda_status(e);
}

int ss_reorder(const ss_reorder_args* a, void* stream) {
  if (a == nullptr) return SS_ERR_INVALID;
  if (a->batch < 0 || a->beams < 1 || a->count < 0) return SS_ERR_INVALID;
  if (a->beams > SS_MAX_BEAMS || a->count > SS_MAX_REORDER || a->batch > 65535) return SS_ERR_UNSUPPORTED;
  if (a->batch == 0 || a->count == 0) return SS_OK;
  if (!a->parents || (a->batch > 1 && a->parents_batch_stride < a->beams)) return SS_ERR_INVALID;
  ReorderK P;
  P.a = *a;
  P.first[0] = 0;
  for (int i = 0; i < a->count; ++i) {
    const int64_t n = a->row_bytes[i];
    if (n < 0 || n % 4 || (n > 0 && (!a->data[i] || (reinterpret_cast<uintptr_t>(a->data[i]) & 3)))) return SS_ERR_INVALID;
    const bool wide = n % 16 == 0 && (reinterpret_cast<uintptr_t>(a->data[i]) & 15) == 0;
    P.first[i + 1] = P.first[i] + ((wide ? n / 16 : n / 4) + 255) / 256;
  }
  P.status = device_status_word();
  if (P.first[a->count] == 0) return SS_OK;
  const dim3 grid((unsigned)std::min<int64_t>(P.first[a->count], std::max<int64_t>(1, 16 * 148 / a->batch)),
                  (unsigned)a->batch);
  cudaStream_t st = (cudaStream_t)stream;
  if (a->beams <= 4) return record_cuda_status(launch_dependent(reorder_kernel<4>, grid, 256, P, st));
  if (a->beams <= 8) return record_cuda_status(launch_dependent(reorder_kernel<8>, grid, 256, P, st));
  if (a->beams <= 16) return record_cuda_status(launch_dependent(reorder_kernel<16>, grid, 256, P, st));
  return record_cuda_status(launch_dependent(reorder_kernel<32>, grid, 256, P, st));
}

}  // extern "C"
