// Linear attention on the 5th-generation tensor cores (tcgen05), for 16-bit I/O: one run of the
// recurrence (ss_linear.cuh) with chunks of 128 tokens.
//
// One CTA walks the chunks of a segment of one (batch row, head) for 64 value columns.  Per chunk:
//
//   S   = Q K^T                 128 x 128 x dk    operands as TMA wrote them (K-major, 128-byte swizzle)
//   P   = S * e^{G_i - G_j}     masked, rounded to 16 bits into TMEM, the A operand of the next product
//   Oa  = P V                   128 x 64 x 128    V as the MN-major B operand
//   Oi  = Q Hhi [+ Q Hlo]       128 x 64 x dk     the state before the chunk, in one or two 16-bit parts
//   L   = K^T V'hi + K^T V'lo   dk x 64 x 128     V' = e^{T - G_j} v_j in two or three parts; K as MN-major A
//   o   = scale (e^{G_i} Oi + Oa),   H <- e^T H + L   (H in fp32 registers, one row a thread)
//
// Rounding: Q, K and V enter as they are.  Each of an output's two sums has one factor rounded to 16 bits
// (half a step): the weighted scores P, and the state H.  An output is rounded to the same type anyway, so
// its error grows by at most sqrt 2.  The weighted values are split: hi + lo keeps 16 (bf16) or 22 (fp16)
// bits, since their rounding would spread to every later token and to the fp32 final state.  Where the dot
// products for the decays' gradient are wanted, H is split as well: the sums of q . dq - k . dk telescope
// only as far as both runs round the same P alike and nothing else.
// fp16 has a mantissa to spare and no range: its weighted scores are scaled by a power of two per row (from a
// bound, the row's largest |q| times the chunk's largest |k| times dk), V' and H by one per chunk (from their
// largest value), which the outputs and the state take back; bf16 needs none of that.
//
// What bounds it: neither memory nor the tensor cores, but the hand-overs between the roles.  A chunk with keys
// of 64 takes about 2.3 us a CTA (a gradient: 4400 cycles, of them 4000 in the warps that make the outputs),
// its products 1500 cycles; a load that was issued early arrives after 3000.  All 19 warps get 96 registers, which
// is too few for the outputs and the state: every instance spills, 136 - 320 bytes stored and 200 - 448 loaded, most
// of it in the gradients' (outputs with their dot products, on the chain).  Measured (kernels, cold L2):
//   8 x 2048 tokens, 24 heads of 64 x 64, bf16       73 us forward (201 MB, 2.7 TB/s), 228 us backward
//   1 x 16384 tokens, 16 heads of 128 x 128, bf16    153 us forward (268 MB, 1.8 TB/s), 170 with the final state
//   4 x 1999 tokens, 16 heads, 4 of keys, fp16       89 us forward, 300 us backward
// Tried and slower: the outputs of gradients shared with the scores' warps (273 against 250 us: a chunk's scores
// then wait for the outputs before them), 32 columns of outputs at a time (295 us: it spills more).
// Two value tiles of one head run side by side, so keys and queries come from L2 the second time.
// Roles (19 warps): 0-3 scores, 4-7 weighted values, 8-11 outputs, 12-15 state, 16 loads, 17 matrix
// instructions, 18 decays.  The only chain from chunk to chunk is H: L -> state warps -> Q H.
#pragma once
#include "ss_linear.cuh"

namespace ssb {

constexpr int kTcC = 128;   // tokens of a chunk
constexpr int kTcN = 64;    // value columns of a CTA
// log decays below this are a reset: e^-88 lies below fp32's normal numbers, and ex2 flushes it to zero
constexpr float kTcReset = -88.f;
// The decays of a stage's chunk, from sums in 64 bits.  Sums of log decays grow with the chunk, and their
// differences, which the weights are made of, keep only the digits that fp32 leaves them; and where the forward
// and the reverse run are left other digits, a score next to a rounding border rounds apart, and the decays'
// gradient, a difference of the two runs, keeps that.  So blocks of 32 tokens count for themselves, and both runs
// form a pair's weight from the same numbers.  With z the sum from a token's block's start to it, t the block's sum
// and s = t - z what follows the token in it (all times log2 e):
//   X        [128]  -z, reverse z: the weight of a pair in one block is 2^{X_col - X_row}, the same bits either way
//   factor   [128]  2^s, reverse 2^z: of a column towards the border of its block on the side of the rows that use it
//   border   [4][4] row block w, column block x: E = 2^(sums of the blocks between them); a pair's weight is
//                   (2^z E) 2^s, reverse (2^s E) 2^z: the same bits for neighbours, whose E is 1.  On the diagonal
//                   the sum of the blocks before w (reverse: behind), which with z (s) is an output's.  Reverse
//                   keeps t of block w in the unused half, at dec_own(w)
//   update   [4]    what a block's factors are multiplied with to weight the update of the state
//   rest     [128]  s - (t - z) in fp32, 8 bits of it, in units that t gives: s where z alone is at hand
// 32 resets in one block leave X half a step of 2^-13, 2^-12.5 of a weight at most: below half a step of fp16.
// Against one fp32 sum a token (1 % faster): the error of dlog_decay over 2600 tokens of log decays around -3, in
// its norm per head, falls from 2.2e-2 to 3.1e-3 (bf16) and from 3.5e-3 to 3.3e-4 (fp16).
constexpr int kDecFactor = kTcC, kDecBorder = 2 * kTcC, kDecUpdate = kDecBorder + 16, kDecRest = kDecUpdate + 4,
              kDecFloats = kDecRest + kTcC / 4;
__device__ __forceinline__ int dec_own(int w) { return kDecBorder + (w < 3 ? 4 * w + 4 : 13); }
constexpr int kTcThreads = 19 * 32;
constexpr uint32_t kBox = kTcC * 128;  // one TMA box: 128 rows of 128 bytes

struct LinTcK {
  LinK k;
  int pass0, tiles, parts;  // first pass of the launch, value tiles of its widest, passes x tiles
  int* status;
  long long wait_limit;
  alignas(64) CUtensorMap map[kLinMaxPasses][4];  // q, k, v, o of each pass
};

// ---------------------------------------------------------------------------------------- PTX
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z), "r"(w), "r"(src)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// every store of this thread has read its shared memory
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// one lane of a converged warp, in the form the compiler knows to be one lane: operands of the
// instructions under it go to uniform registers without a loop over lanes
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Operand descriptors: the low word holds the address (and the distance of 64-wide groups), the high word
// is the same for all of them (8-row groups 1024 bytes apart, 128-byte swizzle)
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n setp.ne.u32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
               "r"((uint32_t)add), "n"(kDescHi)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 y;\n mov.b64 y, {%2, %5};\n setp.ne.u32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
               "r"((uint32_t)add), "n"(kDescHi)
               : "memory");
}
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// low word of a shared-memory operand's descriptor: K-major (rows of 64 elements along K) or MN-major (rows
// of 64 elements along M or N, one K a row; `lead` bytes between groups of 64)
__device__ __forceinline__ uint32_t desc_of(uint32_t addr, uint32_t lead) { return (addr >> 4) | ((lead >> 4) << 16); }
template <typename IT>
__device__ __forceinline__ constexpr uint32_t idesc_of(int m, int n, bool a_mn, bool b_mn) {
  const uint32_t f = std::is_same<IT, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

template <typename IT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<IT, __nv_bfloat16>::value) {
    __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&p);
  } else {
    __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&p);
  }
}
template <typename IT>
__device__ __forceinline__ float2 unpack2(uint32_t p) {
  if constexpr (std::is_same<IT, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<__half2*>(&p));
}
// 8 values of a row split into hi + lo [+ what is left] and stored at 16-byte chunk j of row r of swizzled tiles
template <typename IT>
__device__ __forceinline__ void store_split(unsigned char* hi, unsigned char* lo, unsigned char* rest, int r, int j,
                                            const float (&v)[8]) {
  uint32_t h[4], l[4], t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = pack2<IT>(v[2 * i], v[2 * i + 1]);
    const float2 d = fma2(unpack2<IT>(h[i]), f2(-1.f), make_float2(v[2 * i], v[2 * i + 1]));
    l[i] = pack2<IT>(d.x, d.y);
    if (rest) {
      const float2 e = fma2(unpack2<IT>(l[i]), f2(-1.f), d);
      t[i] = pack2<IT>(e.x, e.y);
    }
  }
  const int at = r * 128 + ((j ^ (r & 7)) << 4);
  *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  if (rest) *reinterpret_cast<uint4*>(rest + at) = make_uint4(t[0], t[1], t[2], t[3]);
}

// Shared memory: stages of Q, K, V as TMA writes them; V' (hi, lo); H (hi, lo); the output tile on its way to
// the TMA store; per stage the decays; barriers.
// Wide heads have room for two stages and none for the output tile, which takes its chunk's V (needed later
// in the stage's next chunk than Q and K).
constexpr uint32_t kBarBytes = 352;

template <int DK>
struct TcShape {
  static constexpr int kBoxes = DK / 64;
  static constexpr int kStages = DK == 128 ? 2 : 3;
  static constexpr bool kOwnOut = DK == 64;
  static constexpr uint32_t kStageBytes = (2 * kBoxes + 1) * kBox;
  static constexpr uint32_t kVAt = 2 * kBoxes * kBox;
  static constexpr uint32_t kVp = kStages * kStageBytes;
  static constexpr uint32_t kH = kVp + 2 * kBox;
  static constexpr uint32_t kOut = kH + 2 * DK * 128;
  static constexpr uint32_t kDecStage = kDecFloats * 4;
  static constexpr uint32_t kDec = kOut + (kOwnOut ? kBox : 0);
  static constexpr uint32_t kBars = kDec + kStages * kDecStage;
  static constexpr uint32_t kBytes = kBars + kBarBytes + 256;  // and the rows' exponents (fp16)
};

struct TcBars {
  uint64_t full[3], empty[3], v_empty[3];
  uint64_t s_full[2], p_full[2];
  uint64_t vp_full[2], vp_empty[2], l_full, l_empty, h_full, h_empty, o_full[2], o_empty[2], drain;
  float total[3];  // e^T of the stage's chunk
  uint32_t tmem;
  int abort;
  // fp16: largest values of a chunk found by four warps, and the exponents they give
  uint64_t max_full[3];
  uint32_t max_of[3][4];
  int v_exp[4], h_exp[4];
};

// TMEM columns: two score buffers (the weighted scores overwrite the first half of theirs, their product
// with V the second), two of Q H, L of the high and of the low parts
constexpr uint32_t kTmS = 0, kTmOa = 64, kTmOi = 256, kTmL = 384, kTmCols = 512;

// try_wait that may suspend the thread for up to ~1 ms instead of coming back at once: a waiting warp
// that polls takes issue slots from the ones that work
__device__ __forceinline__ bool mbar_try_wait_long(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

// a few tens of tries in a loop of four instructions: what a waiting warp issues, the others cannot
__device__ __forceinline__ bool mbar_try_wait_often(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, 0;\n"
      "again:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n @p bra over;\n add.u32 n, n, 1;\n"
      " setp.lt.u32 q, n, 64;\n @q bra again;\n"
      "over:\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

// the part of a wait that is not over at once; false: it gave up, here or in another role
__device__ __noinline__ bool tc_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort, long long limit, int* status) {
  const long long t0 = clock64();
  while (limit == 0 || !mbar_try_wait_often(bar, parity)) {
    if (*abort) return false;
    if (limit == 0 || clock64() - t0 > limit) {
      *abort = 1;
      if (status) atomicOr(status, kStatusTimeout);
      return false;
    }
  }
  return true;
}

// A limit of 0 makes the first wait for a stage a single probe (a choice at every wait cost 5 % of a forward)
__device__ __noinline__ bool tc_first_wait(uint64_t* bar, volatile int* abort, long long limit, int* status) {
  if (limit != 0 || __all_sync(0xffffffffu, mbar_test_wait(bar, 0))) return true;
  return tc_wait_slow(bar, 0, abort, 0, status);
}

// exponent of the power of two that brings values up to m to just below 2^15 (0 where there is nothing to bring)
__device__ __forceinline__ int half_exp(float m) {
  const int e = (int)(__float_as_uint(m) >> 23) & 255;
  return e == 0 || e == 255 ? 0 : max(-100, min(100, 127 + 14 - e));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// largest magnitude of a packed row's words (fp16 only)
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, const uint4& q) {
  auto two = [](uint32_t a, uint32_t b) {
    const __half2 x = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&x);
  };
  m = two(m, q.x & 0x7fff7fffu);
  m = two(m, q.y & 0x7fff7fffu);
  m = two(m, q.z & 0x7fff7fffu);
  return two(m, q.w & 0x7fff7fffu);
}
__device__ __forceinline__ float max_of2(uint32_t m) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
  return fmaxf(f.x, f.y);
}

// 2^-29 of the power of two below |t|, and its inverse: the unit of the rests of a block whose sum is t
__device__ __forceinline__ float2 rest_unit(float t) {
  const uint32_t e = max((__float_as_uint(t) >> 23) & 255u, 64u);
  return make_float2(__uint_as_float((e - 29u) << 23), __uint_as_float((283u - e) << 23));
}
// s = t - z from its three parts
__device__ __forceinline__ float block_rest(float t, float z, int rest) { return fmaf((float)rest, rest_unit(t).x, t - z); }

// What a run writes: the segments' own states; outputs; outputs in parts or with their dot products (gradients
// of q and k); outputs and a final state that is returned
enum { kTcState = 0, kTcOut = 1, kTcGrad = 2, kTcOutState = 3 };

template <typename IT, int DK, int MODE>
__device__ __forceinline__ void linear_tc_run(const LinTcK& P, int pass, int tile, int where, unsigned char* smem) {
  using S = TcShape<DK>;
  constexpr bool STATE_ONLY = MODE == kTcState;
  constexpr bool split_h = MODE == kTcGrad;  // H enters Q H in two parts
  // bf16 states that leave the kernel: V' in three parts (24 bits; two are good to 2.4e-6 of a state's norm,
  // three to 2e-7), the third where the output tile would go
  constexpr bool third = std::is_same<IT, __nv_bfloat16>::value && (MODE == kTcState || MODE == kTcOutState);
  constexpr uint32_t kThird = STATE_ONLY ? S::kH : S::kOwnOut ? S::kOut : S::kH + DK * 128;
  // buffers of V': a state's run, which loads no Q, keeps a second one where the stages' Q would be (its parts
  // one after the other with wide keys, a stage apart with narrow ones)
  constexpr int kVps = STATE_ONLY ? 2 : 1;
  constexpr uint32_t kVp2Lead = DK == 128 ? kBox : S::kStageBytes, kVp2Third = DK == 128 ? S::kStageBytes : 2 * S::kStageBytes;
  // and its three groups with nothing else to do build V' together, by columns (74 -> 70 us over 16384 tokens of
  // 16 heads of 128 x 128; fp16, with a maximum over all columns to find first: 27 us by one group, 34 by three)
  constexpr bool kShare = STATE_ONLY && std::is_same<IT, __nv_bfloat16>::value;
  TcBars& B = *reinterpret_cast<TcBars*>(smem + S::kBars);
  const LinK& K = P.k;
  const LinPass& A = K.pass[pass];
  const int dk = A.dk, dv = A.dv, n0 = tile * kTcN;
  const int bh = where % (K.batch * K.heads), seg = where / (K.batch * K.heads);
  if (!STATE_ONLY && seg > 0) griddep_wait();  // the first segment needs nothing of the passes before
  if (n0 >= dv || (STATE_ONLY && seg == K.segs - 1)) return;
  const int nv = min(kTcN, dv - n0);
  const int b = bh / K.heads, head = bh % K.heads;
  const int len = K.lens ? max(0, min(K.lens[b], K.seqlen)) : K.seqlen;
  const int n_chunks = (K.seqlen + kTcC - 1) / kTcC, n_live = (len + kTcC - 1) / kTcC;
  const int c0 = seg ? K.seg_first + (seg - 1) * K.seg_chunks : 0,
            c1 = min(seg ? c0 + K.seg_chunks : K.seg_first, n_chunks), cn = min(c1, n_live);
  const bool reverse = A.reverse != 0;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, wg = wid >> 2, row = tid & 127;
  auto first_token = [&](int c) { return (reverse ? n_live - 1 - c : c) * kTcC; };
  auto dec_X = [&](int st) { return reinterpret_cast<float*>(smem + S::kDec + st * S::kDecStage); };
  // from a row's X: z, or in reverse s
  auto dec_row = [&](int st, int w, float xi) {
    const float* X = dec_X(st);
    return reverse ? block_rest(X[dec_own(w)], xi, reinterpret_cast<const signed char*>(X + kDecRest)[row]) : -xi;
  };
  const int64_t block = (int64_t)dk * dv;
  // for whole warps: the lanes go on, or give up, together
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_try_wait_long(bar, parity) || tc_wait_slow(bar, parity, &B.abort, P.wait_limit, P.status);
    return __all_sync(0xffffffffu, ok) != 0;
  };

  if (wid == 16 && lane == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&B.full[i], 2);                          // the copies, the decays
      mbar_init(&B.empty[i], STATE_ONLY ? 1 + 4 : 1 + 8);  // the products, the warps that read the decays last
      mbar_init(&B.v_empty[i], STATE_ONLY ? 1 : 1 + 4);    // the products, the output tile that takes V's room
    }
    for (int i = 0; i < 2; ++i) mbar_init(&B.s_full[i], 1), mbar_init(&B.p_full[i], 4);
    for (int i = 0; i < 2; ++i) mbar_init(&B.vp_full[i], kShare ? 12 : 4), mbar_init(&B.vp_empty[i], 1);
    mbar_init(&B.l_full, 1), mbar_init(&B.l_empty, 4);
    mbar_init(&B.h_full, 4), mbar_init(&B.h_empty, 1);
    mbar_init(&B.o_full[0], 1), mbar_init(&B.o_full[1], 1), mbar_init(&B.o_empty[0], 4), mbar_init(&B.o_empty[1], 4);
    mbar_init(&B.drain, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&B.max_full[i], 4);
      for (int j = 0; j < 4; ++j) B.max_of[i][j] = 0;
    }
    B.abort = 0;
    mbar_fence_init();
  }
  if (wid == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)), "r"(kTmCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tm = B.tmem;
  const uint32_t lanes = tm + ((uint32_t)(wid & 3) << 21);  // this warp's 32 lanes

  // The largest m >= 0 of a chunk over the four warps of group `g`, into *m; false: gave up.  Slots go round:
  // who passes the wait of chunk i knows that everyone has read chunk i - 1's.
  auto group_max = [&](int g, int i, float* m) {
    const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(*m));  // order of non-negative floats
    if (lane == 0) {
      atomicMax(&B.max_of[g][i & 3], w);
      mbar_arrive(&B.max_full[g]);
    }
    if (!warp_wait(&B.max_full[g], i & 1)) return false;
    *m = __uint_as_float(*reinterpret_cast<volatile uint32_t*>(&B.max_of[g][i & 3]));
    if ((wid & 3) == 0 && lane == 0) *reinterpret_cast<volatile uint32_t*>(&B.max_of[g][(i + 2) & 3]) = 0;
    return true;
  };
  signed char* row_exp = reinterpret_cast<signed char*>(smem + S::kBars + kBarBytes);  // [2][128]
  constexpr bool kHalf = std::is_same<IT, __half>::value;

  if (wid == 16) {
    // ------------------------------------------------------------ loads
    const int hq = head / A.rq, hk = head / A.rk, hv = head / A.rv;
    const uint32_t base = smem_u32(smem);
    for (int c = c0, i = 0, st = 0, ph = 1; c < cn; ++c, ++i) {
      if (i >= S::kStages && !warp_wait(&B.empty[st], ph)) break;
      const int t0 = first_token(c);
      if (elect_one()) {
        const uint32_t dst = base + st * S::kStageBytes;
        mbar_expect_tx(&B.full[st], (STATE_ONLY ? S::kBoxes + 1 : 2 * S::kBoxes + 1) * kBox);
#pragma unroll
        for (int x = 0; x < S::kBoxes; ++x) {
          if (!STATE_ONLY) tma_load_4d(dst + x * kBox, &P.map[pass][0], x * 64, hq, t0, b, &B.full[st]);
          tma_load_4d(dst + (S::kBoxes + x) * kBox, &P.map[pass][1], x * 64, hk, t0, b, &B.full[st]);
        }
      }
      __syncwarp();
      if (i >= S::kStages && !warp_wait(&B.v_empty[st], ph)) break;
      if (elect_one())
        tma_load_4d(base + st * S::kStageBytes + S::kVAt, &P.map[pass][2], n0, hv, t0, b, &B.full[st]);
      __syncwarp();
      if (++st == S::kStages) st = 0, ph ^= 1;
    }
  } else if (wid == 18) {
    // ------------------------------------------------------------ decays
    constexpr bool bf = std::is_same<IT, __nv_bfloat16>::value;
    uint32_t raw[4];  // 4 tokens a lane of the next chunk, as they are in memory: the loads are under way
    const int64_t g0 = (int64_t)b * K.gb + (int64_t)head * K.gh;
    auto load = [&](int c) {
      const int t = first_token(c) + 4 * lane;
      const int64_t at = g0 + (int64_t)t * K.gl;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        raw[r] = 0u;
        if (t + r < len)
          raw[r] = K.g_f32 ? static_cast<const uint32_t*>(K.g)[at + r * K.gl]
                           : (uint32_t)static_cast<const unsigned short*>(K.g)[at + r * K.gl];
      }
    };
    double seg_total = 0.0;
    if (c0 < cn) load(c0);
    for (int c = c0, i = 0, st = 0, ph = 1; c < cn; ++c, ++i) {
      float g[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (K.g_f32) g[r] = __uint_as_float(raw[r]);
        else if (bf) g[r] = __uint_as_float(raw[r] << 16);
        else g[r] = __half2float(__ushort_as_half((unsigned short)raw[r]));
        g[r] = g[r] < kTcReset ? kTcReset : g[r];  // keeps NaN
      }
      if (c + 1 < cn) load(c + 1);
      // inclusive sums in a block of 8 lanes, in 64 bits, times log2 e
      constexpr double l2e = 1.4426950408889634;
      const double s0 = l2e * (double)g[0], s1 = fma(l2e, (double)g[1], s0), s2 = fma(l2e, (double)g[2], s1),
                   s3 = fma(l2e, (double)g[3], s2);
      double x = s3;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o, 8);
        if ((lane & 7) >= o) x += y;
      }
      double of[4];  // the blocks' sums
#pragma unroll
      for (int r = 0; r < 4; ++r) of[r] = __shfl_sync(0xffffffffu, x, 8 * r + 7);
      const double T = (of[0] + of[1]) + (of[2] + of[3]), before = x - s3, own = __shfl_sync(0xffffffffu, x, 7, 8);
      const double z[4] = {before + s0, before + s1, before + s2, x};
      const float tf = (float)own, unit = rest_unit(tf).y;
      float X[4], factor[4];
      uint32_t rest = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float zf = (float)z[r], s = tf - zf;
        const float q = rintf((float)((own - z[r]) - (double)s) * unit);  // at most 96
        const int qi = (int)fminf(fmaxf(q, -127.f), 127.f);
        rest |= (uint32_t)(qi & 255) << (8 * r);
        X[r] = reverse ? zf : -zf;
        factor[r] = ex2(reverse ? zf : block_rest(tf, zf, qi));
      }
      // lanes 0 - 15: borders, 16 - 19: updates; the sum of blocks `lo` to before `hi`
      const int w = lane >> 2 & 3, c4 = lane & 3;
      const bool upd = lane >= 16, diagonal = w == c4;
      int lo, hi;
      if (upd) lo = reverse ? 0 : c4 + 1, hi = reverse ? c4 : 4;
      else if (!reverse) lo = diagonal ? 0 : c4 + 1, hi = w;
      else if (c4 < w) lo = c4 ? 3 : w - 1, hi = lo + 1;
      else lo = w + 1, hi = diagonal ? 4 : c4;
      double sum = 0.0;
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += r >= lo && r < hi ? of[r] : 0.0;
      const float entry = (float)sum;
      const bool raw = !upd && (diagonal || (reverse && c4 < w));
      seg_total += T;
      if (i >= S::kStages && !warp_wait(&B.empty[st], ph)) break;
      float* xs = dec_X(st);
      *reinterpret_cast<float4*>(xs + 4 * lane) = make_float4(X[0], X[1], X[2], X[3]);
      *reinterpret_cast<float4*>(xs + kDecFactor + 4 * lane) = make_float4(factor[0], factor[1], factor[2], factor[3]);
      reinterpret_cast<uint32_t*>(xs + kDecRest)[lane] = rest;
      if (lane < 20) xs[kDecBorder + lane] = raw ? entry : ex2(entry);
      if (lane == 0) B.total[st] = ex2((float)T);
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.full[st]);
      if (++st == S::kStages) st = 0, ph ^= 1;
    }
    if (STATE_ONLY && tile == 0 && lane == 0)
      K.seg_decay[((int64_t)reverse * K.batch * K.heads + bh) * K.segs + seg] = (float)(seg_total * 0.6931471805599453);
  } else if (wid == 17) {
    // ------------------------------------------------------------ matrix instructions
    const uint32_t base = smem_u32(smem);
    constexpr uint32_t kIdQK = idesc_of<IT>(128, kTcC, false, false), kIdN = idesc_of<IT>(128, kTcN, false, true),
                       kIdL = idesc_of<IT>(128, 2 * kTcN, true, true);
    // descriptors of the first stage; a step of 16 along K is 32 bytes (K-major) or 2048 (MN-major)
    const uint32_t q0 = desc_of(base, 16), kk0 = desc_of(base + S::kBoxes * kBox, 16),
                   km0 = desc_of(base + S::kBoxes * kBox, kBox), v0 = desc_of(base + S::kVAt, kBox),
                   vp0 = desc_of(base + S::kVp, kBox), h0 = desc_of(base + S::kH, kBox);
    auto scores = [&](int st, int buf) {
      const uint32_t o = st * (S::kStageBytes >> 4);
      if (elect_one()) {
#pragma unroll
        for (int x = 0; x < DK / 16; ++x) {
          const uint32_t at = (x >> 2) * (kBox >> 4) + (x & 3) * 2;
          mma_ss(tm + kTmS + buf * 128, q0 + o + at, kk0 + o + at, kIdQK, x > 0);
        }
        tc_commit(&B.s_full[buf]);
      }
      __syncwarp();
    };
    const int n = cn > c0 && tc_first_wait(&B.full[0], &B.abort, P.wait_limit, P.status) ? cn - c0 : 0;
    for (int i = 0, st = 0, ph = 0; i < n; ++i) {  // ph: the stages' phase
      if (!warp_wait(&B.full[st], ph)) break;
      tc_after();
      if (!STATE_ONLY && i == 0) scores(0, 0);
      // L = K^T [V'hi, V'lo]: a product of 64 columns takes as long as one of 128
      if (!warp_wait(&B.vp_full[kVps == 2 ? i & 1 : 0], (uint32_t)(i / kVps) & 1) || (i > 0 && !warp_wait(&B.l_empty, (i - 1) & 1))) break;
      tc_after();
      const uint32_t o = st * (S::kStageBytes >> 4), vp = kVps == 2 && (i & 1) ? desc_of(base, kVp2Lead) : vp0;
      if (elect_one()) {
#pragma unroll
        for (int x = 0; x < kTcC / 16; ++x) mma_ss(tm + kTmL, km0 + o + x * 128, vp + x * 128, kIdL, x > 0);
        if constexpr (third) {  // onto the low part's columns
          const uint32_t v3 = kVps == 2 && (i & 1) ? desc_of(base + kVp2Third, kBox) : desc_of(base + kThird, kBox);
#pragma unroll
          for (int x = 0; x < kTcC / 16; ++x)
            mma_ss(tm + kTmL + kTcN, km0 + o + x * 128, v3 + x * 128, idesc_of<IT>(128, kTcN, true, true), true);
        }
        tc_commit(&B.vp_empty[kVps == 2 ? i & 1 : 0]);
        tc_commit(&B.l_full);
        if (STATE_ONLY) tc_commit(&B.empty[st]), tc_commit(&B.v_empty[st]);
      }
      __syncwarp();
      const int nst = st + 1 == S::kStages ? 0 : st + 1, nph = nst ? ph : ph ^ 1;
      if constexpr (!STATE_ONLY) {
        // Oi = Q H
        if (!warp_wait(&B.h_full, i & 1)) break;
        tc_after();
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < DK / 16; ++x)
            mma_ss(tm + kTmOi + (i & 1) * kTcN, q0 + o + (x >> 2) * (kBox >> 4) + (x & 3) * 2, h0 + x * 128, kIdN, x > 0);
          if constexpr (split_h) {
#pragma unroll
            for (int x = 0; x < DK / 16; ++x)
              mma_ss(tm + kTmOi + (i & 1) * kTcN, q0 + o + (x >> 2) * (kBox >> 4) + (x & 3) * 2,
                     h0 + (DK / 16 + x) * 128, kIdN, true);
          }
          tc_commit(&B.h_empty);
        }
        __syncwarp();
        // the next chunk's scores, into the buffer whose outputs were read (o_empty; those of Q H before them
        // as well): now if chunk and buffer are there, else after this chunk's last product, which must not
        // wait for them
        bool ahead = i + 1 < n && __all_sync(0xffffffffu, mbar_test_wait(&B.full[nst], nph) &&
                                                              (i == 0 || mbar_test_wait(&B.o_empty[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1)));
        if (ahead) {
          tc_after();
          scores(nst, (i + 1) & 1);
        }
        // Oa = P V
        if (!warp_wait(&B.p_full[i & 1], (uint32_t)(i >> 1) & 1)) break;
        tc_after();
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < kTcC / 16; ++x)
            mma_ts(tm + kTmOa + (i & 1) * 128, tm + kTmS + (i & 1) * 128 + x * 8, v0 + o + x * 128, kIdN, x > 0);
          tc_commit(&B.o_full[i & 1]);
          tc_commit(&B.empty[st]);
          tc_commit(&B.v_empty[st]);
        }
        __syncwarp();
        if (!ahead && i + 1 < n) {
          if (!warp_wait(&B.full[nst], nph) || (i > 0 && !warp_wait(&B.o_empty[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1))) break;
          tc_after();
          scores(nst, (i + 1) & 1);
        }
      }
      st = nst;
      ph = nph;
    }
    // every product has ended before the CTA gives up its memory
    if (elect_one()) tc_commit(&B.drain);
    __syncwarp();
    const long long t0 = clock64();
    while (!mbar_try_wait(&B.drain, 0) && clock64() - t0 < kWaitCycles) {
    }
    __syncwarp();
  } else if (!STATE_ONLY && wg == 0) {
    // ------------------------------------------------------------ weighted scores
    if constexpr (!STATE_ONLY) {
      const int w = wid & 3;
      const uint32_t diag = reverse ? 0xffffffffu << lane : 0xffffffffu >> (31 - lane);  // columns kept of the lane's row
      for (int c = c0, i = 0, st = 0, ph = 0; c < cn; ++c, ++i) {
        const int m = min(kTcC, len - first_token(c));
        if (!warp_wait(&B.full[st], ph) || !warp_wait(&B.s_full[i & 1], (uint32_t)(i >> 1) & 1)) break;
        float pw = 1.f;  // fp16: the row's scale
        if constexpr (kHalf) {
          uint32_t qm = 0, km = 0;
#pragma unroll 1
          for (int j = 0; j < DK / 8; ++j) {
            const unsigned char* at = smem + st * S::kStageBytes + (j >> 3) * kBox + row * 128 + (j & 7) * 16;
            qm = max_abs2(qm, *reinterpret_cast<const uint4*>(at));
            km = max_abs2(km, *reinterpret_cast<const uint4*>(at + S::kBoxes * kBox));
          }
          float k = row < m ? max_of2(km) : 0.f;
          if (!group_max(0, i, &k)) break;
          const int e = half_exp(max_of2(qm) * k * DK);
          row_exp[(i & 1) * 128 + row] = (signed char)e;
          pw = pow2(e);
        }
        tc_after();
        const float* X = dec_X(st);
        const float xi = X[row];
        // the row's part of its weights off the diagonal
        const float own = pw * ex2(dec_row(st, w, xi));
        const uint32_t sp = lanes + kTmS + (i & 1) * 128;
        // 32 columns at a time.  P's columns x .. x + 31 land on S's columns x / 2 .., always behind
        // what is still to be read; blocks on the far side of the diagonal are zero.  Off the diagonal one
        // exponential a row, and the columns' factors from the warp of the decays
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          uint32_t p[16];
          if (reverse ? x >= w : x <= w) {
            float s[32];
            tmem_ld32(sp + x * 32, s);
            if (x != w) {
              const float2 rf = f2(own * X[kDecBorder + 4 * w + x]);
              const float* cf = X + kDecFactor + x * 32;
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 f = *reinterpret_cast<const float4*>(cf + j);
                const float2 e0 = mul2(make_float2(s[j], s[j + 1]), mul2(rf, make_float2(f.x, f.y)));
                const float2 e1 = mul2(make_float2(s[j + 2], s[j + 3]), mul2(rf, make_float2(f.z, f.w)));
                s[j] = e0.x, s[j + 1] = e0.y, s[j + 2] = e1.x, s[j + 3] = e1.y;
              }
            } else {
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 xj = *reinterpret_cast<const float4*>(X + x * 32 + j);
                const float x4[4] = {xj.x, xj.y, xj.z, xj.w};
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float e = s[j + r] * (kHalf ? pw * ex2_ordered(x4[r] - xi) : ex2_ordered(x4[r] - xi));
                  s[j + r] = diag & (1u << (j + r)) ? e : 0.f;
                }
              }
            }
            if (reverse && m < kTcC) {  // columns behind the row's end hold anything
#pragma unroll
              for (int j = 0; j < 32; ++j) s[j] = x * 32 + j < m ? s[j] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) p[j] = pack2<IT>(s[2 * j], s[2 * j + 1]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) p[j] = 0u;
          }
          tmem_st16(sp + x * 16, p);
        }
        tc_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[i & 1]);
        if (++st == S::kStages) st = 0, ph ^= 1;
      }
    }
  } else if (kShare ? wg < 3 : wg == 1) {
    // ------------------------------------------------------------ weighted values
    const int j0 = kShare ? 3 * wg : 0, j1 = kShare ? min(j0 + 3, 8) : 8;
    if constexpr (third && !STATE_ONLY) asm volatile("bar.sync 1, 256;" ::: "memory");  // the state has left the room
    for (int c = c0, i = 0, st = 0, ph = 0; c < cn; ++c, ++i) {
      const int m = min(kTcC, len - first_token(c));
      if (!warp_wait(&B.full[st], ph)) break;
      unsigned char* k = smem + st * S::kStageBytes + S::kBoxes * kBox + row * 128;
      unsigned char* v = smem + st * S::kStageBytes + S::kVAt + row * 128;
      if (row >= m) {  // behind the row's end: whatever was read there must not meet a product
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int x = 0; x < S::kBoxes; ++x) *reinterpret_cast<uint4*>(k + x * kBox + j * 16) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(v + j * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      __syncwarp();
      float wv = dec_X(st)[kDecFactor + row] * dec_X(st)[kDecUpdate + (row >> 5)];
      int v_exp = 0;
      if constexpr (kHalf) {
        uint32_t vm = 0;
#pragma unroll 1
        for (int j = 0; j < 8; ++j) vm = max_abs2(vm, *reinterpret_cast<const uint4*>(v + j * 16));
        float x = wv * max_of2(vm);
        if (!group_max(1, i, &x)) break;
        v_exp = half_exp(x);
        wv *= pow2(v_exp);
      }
      const float2 w = f2(wv);
      // the product over the buffer has ended
      if (i >= kVps && !warp_wait(&B.vp_empty[kVps == 2 ? i & 1 : 0], (uint32_t)(i / kVps - 1) & 1)) break;
      if (kHalf && row == 0) *reinterpret_cast<volatile int*>(&B.v_exp[i & 3]) = v_exp;
      const bool second = kVps == 2 && (i & 1);
      unsigned char *vp = second ? smem : smem + S::kVp, *lo = vp + (second ? kVp2Lead : kBox),
                    *rest = third ? smem + (second ? kVp2Third : kThird) : nullptr;
#pragma unroll 2
      for (int j = j0; j < j1; ++j) {
        const uint4 q = *reinterpret_cast<const uint4*>(v + ((j ^ (row & 7)) << 4));
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
        float x[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 f = mul2(w, unpack2<IT>(u[r]));
          x[2 * r] = f.x;
          x[2 * r + 1] = f.y;
        }
        store_split<IT>(vp, lo, rest, row, j, x);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.vp_full[kVps == 2 ? i & 1 : 0]);
      if (++st == S::kStages) st = 0, ph ^= 1;
    }
  } else if (!STATE_ONLY && wg == 2) {
    // ------------------------------------------------------------ outputs
    if constexpr (!STATE_ONLY) {
      const bool o_f32 = MODE == kTcGrad && A.o_f32;
      const int w4 = wid & 3;
      // wide heads: the room of H's low part where that is not used; fp32 tiles, twice as large, take Q's and K's
      const bool own_out = (S::kOwnOut || !split_h) && !third && !o_f32;
      const IT* p_at = A.dot ? static_cast<const IT*>(A.p) + (int64_t)b * A.pb + (int64_t)(head / A.rp) * A.ph + n0 : nullptr;
      float* dot_at = MODE == kTcGrad && A.dot ? A.dot + (((int64_t)tile * K.batch + b) * K.heads + head) * K.seqlen : nullptr;
      const float2 sc = f2(A.scale);
      // the rows of p that go with a chunk's outputs, 8 lanes a row: loaded a chunk ahead, then passed through
      // shared memory, since a lane that read its own row would touch 32 lines an instruction
      uint4 pq[8];
      auto load_p = [&](int c) {
        const int t0 = first_token(c), m = min(kTcC, len - t0);
        const IT* p = p_at + (int64_t)(t0 + w4 * 32 + (lane >> 3)) * A.pl + (lane & 7) * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          pq[k] = ld_vector(p + (int64_t)4 * k * A.pl, w4 * 32 + 4 * k + (lane >> 3) < m && (lane & 7) * 8 < nv);
      };
      if (dot_at && c0 < cn) load_p(c0);
      for (int c = c0, i = 0, st = 0, ph = 0; c < cn; ++c, ++i) {
        const int t0 = first_token(c), m = min(kTcC, len - t0), t = t0 + row;
        if (!warp_wait(&B.full[st], ph)) break;
        const float2 w = f2(A.scale * ex2(dec_X(st)[kDecBorder + 5 * w4] + dec_row(st, w4, dec_X(st)[row])));
        const bool on = row < m;
        __syncwarp();
        if (lane == 0) {
          if (!o_f32) mbar_arrive(&B.empty[st]);
          if (own_out) mbar_arrive(&B.v_empty[st]);
        }
        if (!warp_wait(&B.o_full[i & 1], (uint32_t)(i >> 1) & 1)) break;
        tc_after();
        float2 wi = w, wa = sc;
        if constexpr (kHalf) {
          wi = mul2(wi, f2(pow2(-*reinterpret_cast<volatile int*>(&B.h_exp[i & 3]))));
          wa = mul2(wa, f2(pow2(-row_exp[(i & 1) * 128 + row])));
        }
        const uint32_t tile_at = own_out ? (S::kOwnOut ? S::kOut : S::kH + DK * 128) : st * S::kStageBytes + (o_f32 ? 0 : S::kVAt);
        if (own_out) {
          if (elect_one()) tma_store_read();  // the tile before has left
          __syncwarp();
        }
        unsigned char* out = smem + tile_at + row * 128;
        const unsigned char* prow = o_f32 ? smem + st * S::kStageBytes + S::kVAt + row * 128 : out;  // V has been used
        if (dot_at) {
          unsigned char* to = const_cast<unsigned char*>(prow) - row * 128;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = w4 * 32 + 4 * k + (lane >> 3);
            *reinterpret_cast<uint4*>(to + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = pq[k];
          }
          __syncwarp();
          if (c + 1 < cn) load_p(c + 1);
        }
        float2 dot = f2(0.f);
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          float o[16], oa[16];
          tmem_ld16(lanes + kTmOi + (i & 1) * kTcN + x * 16, o);
          tmem_ld16(lanes + kTmOa + (i & 1) * 128 + x * 16, oa);
          uint4 q0, q1;
          if (dot_at) {
            q0 = *reinterpret_cast<const uint4*>(prow + (((2 * x) ^ (row & 7)) << 4));
            q1 = *reinterpret_cast<const uint4*>(prow + (((2 * x + 1) ^ (row & 7)) << 4));
          }
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 r = fma2(wi, make_float2(o[j], o[j + 1]), mul2(wa, make_float2(oa[j], oa[j + 1])));
            o[j] = on ? r.x : 0.f, o[j + 1] = on ? r.y : 0.f;
          }
          if (o_f32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(out + (x >> 1) * kBox + ((((x & 1) * 4 + j) ^ (row & 7)) << 4)) =
                  make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              *reinterpret_cast<uint4*>(out + (((2 * x + j) ^ (row & 7)) << 4)) =
                  make_uint4(pack2<IT>(o[8 * j], o[8 * j + 1]), pack2<IT>(o[8 * j + 2], o[8 * j + 3]),
                             pack2<IT>(o[8 * j + 4], o[8 * j + 5]), pack2<IT>(o[8 * j + 6], o[8 * j + 7]));
          }
          if (dot_at) {
            const uint32_t u[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) dot = fma2(make_float2(o[2 * j], o[2 * j + 1]), unpack2<IT>(u[j]), dot);
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&B.o_empty[i & 1]);
          if (o_f32) mbar_arrive(&B.v_empty[st]);
        }
        fence_async_smem();
        __syncwarp();
        if (elect_one()) {
          if (t0 + w4 * 32 < K.seqlen) {
            const uint32_t src = smem_u32(smem) + tile_at + w4 * 32 * 128;
            tma_store_4d(&P.map[pass][3], src, n0, head, t0 + w4 * 32, b);
            if (o_f32 && n0 + 32 < dv) tma_store_4d(&P.map[pass][3], src + kBox, n0 + 32, head, t0 + w4 * 32, b);
          }
          if (own_out) {
            tma_store_commit();
          } else {
            tma_store_commit();
            tma_store_read();
            mbar_arrive(o_f32 ? &B.empty[st] : &B.v_empty[st]);
          }
        }
        __syncwarp();
        if (dot_at && t < K.seqlen) dot_at[t] = on ? dot.x + dot.y : 0.f;
        if (++st == S::kStages) st = 0, ph ^= 1;
      }
      if (elect_one()) tma_store_read();
      __syncwarp();
      auto zero_row = [&](int t) {
        const int es = o_f32 ? 4 : 2;
        char* o = static_cast<char*>(A.o) + ((int64_t)b * A.ob + (int64_t)t * A.ol + (int64_t)head * A.oh + n0) * es;
#pragma unroll 1
        for (int j = 0; j < nv * es; j += 16) *reinterpret_cast<uint4*>(o + j) = make_uint4(0, 0, 0, 0);
        if (dot_at) dot_at[t] = 0.f;
      };
      for (int c = max(cn, c0); c < c1; ++c)  // chunks behind the row's end
        if (c * kTcC + row < K.seqlen) zero_row(c * kTcC + row);
    }
  } else if (wg == 3) {
    // ------------------------------------------------------------ state: row `row` of H
    // Rows enter and leave the registers through the room of the 16-bit halves (256 bytes a row), each
    // warp its own: short loops, and a warp's lanes side by side along a row in memory
    float h[kTcN];
    float* rows = reinterpret_cast<float*>(smem + S::kH) + (wid & 3) * 32 * kTcN;
    const int r0 = (wid & 3) * 32, rn = min(32, dk - r0);  // this warp's rows; <= 0: none
    const bool from = !STATE_ONLY && r0 < DK && (seg > 0 || A.s_in != nullptr);  // else from zeros
    if (from) {
      // 8 loads under way at a time
      auto each = [&](auto&& f) {
#pragma unroll 1
        for (int e0 = lane; e0 < 32 * kTcN; e0 += 8 * 32) {
          float x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int e = e0 + 32 * u, r = e / kTcN, j = e % kTcN;
            x[u] = r < rn && j < nv ? f(r, j) : 0.f;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int e = e0 + 32 * u;
            rows[e] = x[u];
          }
        }
      };
      if (seg > 0) {  // folded from the initial state and the segments before
        const float* s0 = A.sum + ((int64_t)bh * K.segs + seg) * block + (int64_t)r0 * dv + n0;
        each([&](int r, int j) { return s0[(int64_t)r * dv + j]; });
      } else {
        const float* s0 = A.s_in + bh * block + (int64_t)r0 * A.s_row + (int64_t)n0 * A.s_col;
        each([&](int r, int j) { return A.s_in_scale * s0[(int64_t)r * A.s_row + (int64_t)j * A.s_col]; });
      }
      __syncwarp();
    }
#pragma unroll
    for (int j = 0; j < kTcN; j += 4) {
      const float4 x = from ? *reinterpret_cast<const float4*>(rows + lane * kTcN + j) : make_float4(0.f, 0.f, 0.f, 0.f);
      h[j] = x.x, h[j + 1] = x.y, h[j + 2] = x.z, h[j + 3] = x.w;
    }
    // the halves of one warp lie in the rows of others, and so may V's third part
    if constexpr (!STATE_ONLY) asm volatile("bar.sync 1, %0;" ::"n"(third ? 256 : 128) : "memory");
    unsigned char* hh = smem + S::kH;
    auto publish = [&](int i) {
      float2 hw = f2(1.f);
      if constexpr (kHalf) {
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < kTcN; ++j) x = fmaxf(x, fabsf(h[j]));
        if (row >= dk) x = 0.f;
        if (!group_max(2, i, &x)) return false;
        const int e = half_exp(x);
        hw = f2(pow2(e));
        if (row == 0) *reinterpret_cast<volatile int*>(&B.h_exp[i & 3]) = e;
      }
      if (row < DK) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float x[8];
#pragma unroll
          for (int r = 0; r < 8; r += 2) {
            const float2 t = kHalf ? mul2(hw, make_float2(h[8 * j + r], h[8 * j + r + 1]))
                                   : make_float2(h[8 * j + r], h[8 * j + r + 1]);
            x[r] = t.x, x[r + 1] = t.y;
          }
          if constexpr (split_h) {
            store_split<IT>(hh, hh + DK * 128, nullptr, row, j, x);
          } else {
            *reinterpret_cast<uint4*>(hh + row * 128 + ((j ^ (row & 7)) << 4)) =
                make_uint4(pack2<IT>(x[0], x[1]), pack2<IT>(x[2], x[3]), pack2<IT>(x[4], x[5]), pack2<IT>(x[6], x[7]));
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.h_full);
      return true;
    };
    for (int c = c0, i = 0, st = 0, ph = 0; c < cn; ++c, ++i) {
      if (!STATE_ONLY) {
        if (i > 0 && !warp_wait(&B.h_empty, (i - 1) & 1)) break;
        if (!publish(i)) break;
      }
      if (!warp_wait(&B.full[st], ph)) break;
      const float d = *reinterpret_cast<volatile float*>(&B.total[st]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.empty[st]);
      if (!warp_wait(&B.l_full, i & 1)) break;
      tc_after();
      const float2 lw = f2(kHalf ? pow2(-*reinterpret_cast<volatile int*>(&B.v_exp[i & 3])) : 1.f);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float l[16], lo[16];
        tmem_ld16(lanes + kTmL + x * 16, l);
        tmem_ld16(lanes + kTmL + kTcN + x * 16, lo);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          float2 t = add2(make_float2(l[j], l[j + 1]), make_float2(lo[j], lo[j + 1]));
          if (kHalf) t = mul2(lw, t);
          const float2 r = fma2(f2(d), make_float2(h[x * 16 + j], h[x * 16 + j + 1]), t);
          h[x * 16 + j] = r.x, h[x * 16 + j + 1] = r.y;
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.l_empty);
      if (++st == S::kStages) st = 0, ph ^= 1;
    }
    // the last product over V' has ended (l_full): the rows leave through its room
    rows = reinterpret_cast<float*>(smem + S::kVp) + (wid & 3) * 32 * kTcN;
    const bool ok = *reinterpret_cast<volatile int*>(&B.abort) == 0;
    float* to = STATE_ONLY ? A.sum + ((int64_t)bh * K.segs + seg) * block
                           : (A.s_out && seg == K.segs - 1 ? A.s_out + bh * block : nullptr);
    if (to && r0 < DK) {
#pragma unroll
      for (int j = 0; j < kTcN; j += 4)
        *reinterpret_cast<float4*>(rows + lane * kTcN + j) = make_float4(h[j], h[j + 1], h[j + 2], h[j + 3]);
      __syncwarp();
      const float f = STATE_ONLY ? 1.f : A.s_out_scale;
      const int64_t sr = STATE_ONLY ? dv : A.s_row, sc = STATE_ONLY ? 1 : A.s_col;
#pragma unroll 1
      for (int e = lane; e < 32 * kTcN; e += 32) {
        const int r = e / kTcN, j = e % kTcN;
        if (ok && r < rn && j < nv) to[(int64_t)(r0 + r) * sr + (int64_t)(n0 + j) * sc] = f * rows[e];
      }
    }
  }
  tc_before();
  __syncthreads();
  if (B.abort && wid == 16 && lane == 0) {  // copies still in flight land before the memory is given up
    const long long t0 = clock64();
    for (int st = 0; st < S::kStages; ++st)
      for (uint32_t par = 0; par < 2; ++par)
        while (!mbar_try_wait(&B.full[st], par) && clock64() - t0 < kWaitCycles / 8) {
        }
  }
  __syncthreads();
  if (wid == 17) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(kTmCols) : "memory");
  }
}

// Value tiles and runs of one head are neighbours in the grid, so that they share what they read in L2; runs
// with narrow and with wide keys go side by side in one launch.  One kernel a mode: together they spilled and
// fought over the instruction cache (8 x 2048 tokens of 24 heads of 64, gradients: 322 us in one launch, 250 in two).
template <typename IT, int MODE>
__global__ void __launch_bounds__(kTcThreads, 1) linear_tc_kernel(const __grid_constant__ LinTcK P) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const int part = blockIdx.x % P.parts, where = blockIdx.x / P.parts;
  const int pass = P.pass0 + part / P.tiles, tile = part % P.tiles;
  griddep_launch_dependents();
  if (P.k.pass[pass].dk > 64) linear_tc_run<IT, 128, MODE>(P, pass, tile, where, smem);
  else linear_tc_run<IT, 64, MODE>(P, pass, tile, where, smem);
  griddep_wait();  // blocks that had nothing to wait for do not end before the launches ahead of theirs
}

}  // namespace ssb
