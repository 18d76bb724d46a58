// The norm after a block, the block's gate and residual scale, the residual sum and the norm before the next block
// (+ dynamic int8 quantisation of its result) in one pass over the row.
//
//   t  = x * r1 * post_weight            r1 = 1 / sqrt(mean(x^2) + post_eps)
//   r' = residual + (c * gate) * t       residual_out = r' rounded to the type
//   y  = r' * r2 * pre_weight            r2 = 1 / sqrt(mean(r'^2) + pre_eps), from r' before its rounding
//   scale = max|y| / 127, q = rint(y / scale), on y as its type holds it
//
// Everything between the loads and the one rounding of each output is fp32.  Bound by memory: 4 elements of
// traffic for about 15 operations.  A block per row keeps the row in registers through both reductions, so x and
// residual are read once; the two reductions cannot be joined into one pass, because the second norm's sum of
// squares taken from the sums of x^2, x*r and r^2 cancels where the block undoes the residual.  8192 rows of 7168 in bf16:
// 470 MB in 90 to 100 us, 4.7 to 5.2 TB/s; a plain copy of that size moves 5.0 TB/s.
#include "rows.h"

namespace {

struct SandwichArgs {
  const void *x, *residual, *post_w, *pre_w, *gate;
  int64_t ldx, ldr, ldg, ldo;
  int H, gate_mode;
  float post_eps, pre_eps, c;
  void *residual_out, *y;
  int8_t* q;
  float* scale;
};

template <int DT, int THREADS, int MAXV, bool ALIGNED>
__global__ __launch_bounds__(THREADS) void sandwich_norm_kernel(SandwichArgs a) {
  typedef typename Elem<DT>::T ET;
  constexpr int NW = THREADS / WAVE;
  __shared__ float red1[NW], red2[NW];
  __shared__ uint32_t redm[NW];
  const int64_t r = blockIdx.x;
  const int H = a.H, nvec = (H + 7) / 8;
  const ET* xr = (const ET*)a.x + r * a.ldx;
  const ET* rr = (const ET*)a.residual + r * a.ldr;
  const bool wide_gate = a.gate_mode == OMNI_GATE_CHANNEL || a.gate_mode == OMNI_GATE_FULL;
  const ET* gr = (const ET*)a.gate + (a.gate_mode == OMNI_GATE_FULL ? r * a.ldg : 0);
  float s[MAXV][8], d[MAXV][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int vi = threadIdx.x + i * THREADS;
    if (vi < nvec) {
      load8<DT, ALIGNED>(xr, vi, H, s[i]);
      load8<DT, ALIGNED>(rr, vi, H, d[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = ss + s[i][j] * s[i][j];
    }
  }
  const float r1 = 1.0f / sqrtf(block_sum<THREADS>(ss, red1) / (float)H + a.post_eps);
  const float c = a.gate_mode == OMNI_GATE_TOKEN ? a.c * Elem<DT>::cvt(((const ET*)a.gate)[r * a.ldg]) : a.c;
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int vi = threadIdx.x + i * THREADS;
    if (vi < nvec) {
      float w[8];
      load8<DT, ALIGNED>((const ET*)a.post_w, vi, H, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = (s[i][j] * r1) * w[j];
      if (wide_gate) {
        load8<DT, ALIGNED>(gr, vi, H, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = (a.c * w[j]) * s[i][j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = c * s[i][j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] = d[i][j] + s[i][j];
        ss = ss + (vi * 8 + j < H ? s[i][j] * s[i][j] : 0.0f);
      }
      store8<DT, ALIGNED>((ET*)a.residual_out + r * a.ldo, vi, H, s[i]);
    }
  }
  if (a.y == nullptr && a.q == nullptr) return;
  const float r2 = 1.0f / sqrtf(block_sum<THREADS>(ss, red2) / (float)H + a.pre_eps);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int vi = threadIdx.x + i * THREADS;
    if (vi < nvec) {
      float w[8];
      load8<DT, ALIGNED>((const ET*)a.pre_w, vi, H, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] = round_to<DT>((s[i][j] * r2) * w[j]);
        if (ALIGNED || vi * 8 + j < H) m = max(m, abs_bits(s[i][j]));
      }
      if (a.y) store8<DT, ALIGNED>((ET*)a.y + r * H, vi, H, s[i]);
    }
  }
  if (a.q == nullptr) return;
  const float sc = block_absmax<THREADS>(m, redm) / 127.0f;
  if (threadIdx.x == 0) a.scale[r] = sc;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int vi = threadIdx.x + i * THREADS;
    if (vi < nvec) store_q8<ALIGNED>(a.q + r * H, vi, H, s[i], sc);
  }
}

constexpr int SANDWICH_MAX_H = 16384;

// Few rows (up to two per compute unit): 1024 threads, a vector each, which is 5.3 us for one row of 7168 where 256
// threads with four each take 7.8, and 6.6 against 9.6 us for 64 rows of 7680 (what is left is the launch, the way to
// memory and back and the two reductions; weights loaded ahead of them change nothing).  Many rows: 512 threads, 101 us
// for 8192 rows of 7168 against 111 (256) and 116 us (1024).
template <int DT, bool ALIGNED>
int launch_sandwich(const SandwichArgs& a, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)rows);
#define SANDWICH(THREADS, MAXV) \
  hipLaunchKernelGGL((sandwich_norm_kernel<DT, THREADS, MAXV, ALIGNED>), grid, dim3(THREADS), 0, st, a)
  if (a.H <= 8 * 256) SANDWICH(256, 1);
  else if (a.H > 8 * 1024) SANDWICH(1024, 2);
  else if (rows <= 512) SANDWICH(1024, 1);
  else SANDWICH(512, 2);
#undef SANDWICH
  OMNI_CHECK_LAUNCH("sandwich_norm");
  return OMNI_OK;
}

}  // namespace

extern "C" int omni_sandwich_norm(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ld_residual,
                                  const void* post_weight, const void* pre_weight, const void* gate, int gate_mode,
                                  int64_t ld_gate, int64_t rows, int H, float post_eps, float pre_eps,
                                  float residual_scale, void* residual_out, int64_t ld_residual_out, void* y, int8_t* q,
                                  float* scale, void* stream) {
  if (dtype != OMNI_DT_BF16 && dtype != OMNI_DT_F16 && dtype != OMNI_DT_F32)
    OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: unknown dtype %d", dtype);
  if (rows < 0 || H <= 0) OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: bad shape rows=%lld H=%d", (long long)rows, H);
  if (ldx < H || ld_residual < H || ld_residual_out < H)
    OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: a row stride is below H=%d", H);
  if (gate_mode < OMNI_GATE_NONE || gate_mode > OMNI_GATE_FULL) OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: bad gate mode %d", gate_mode);
  if ((gate != nullptr) != (gate_mode != OMNI_GATE_NONE)) OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: gate and gate mode go together");
  if ((gate_mode == OMNI_GATE_TOKEN && ld_gate < 1) || (gate_mode == OMNI_GATE_FULL && ld_gate < H))
    OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: bad row stride %lld of the gate", (long long)ld_gate);
  if (rows == 0) return OMNI_OK;
  if (!x || !residual || !post_weight || !pre_weight || !residual_out) OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: null pointer");
  if ((q == nullptr) != (scale == nullptr)) OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: q and scale go together");
  if (H > SANDWICH_MAX_H) OMNI_FAIL(OMNI_E_UNSUPPORTED, "sandwich_norm: H=%d is above %d", H, SANDWICH_MAX_H);
  if (rows > ROWS_MAX) OMNI_FAIL(OMNI_E_UNSUPPORTED, "sandwich_norm: %lld rows, at most %lld", (long long)rows, (long long)ROWS_MAX);
  const size_t es = dtype == OMNI_DT_F32 ? 4 : 2;
  if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)post_weight | (uintptr_t)pre_weight | (uintptr_t)gate |
       (uintptr_t)residual_out | (uintptr_t)y) % es || (uintptr_t)scale % 4)
    OMNI_FAIL(OMNI_E_INVALID, "sandwich_norm: misaligned pointer");
  const uintptr_t places = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)post_weight | (uintptr_t)pre_weight |
                           (uintptr_t)residual_out | (uintptr_t)y | (uintptr_t)(ldx * es) | (uintptr_t)(ld_residual * es) |
                           (uintptr_t)(ld_residual_out * es) |
                           (gate_mode == OMNI_GATE_CHANNEL || gate_mode == OMNI_GATE_FULL ? (uintptr_t)gate : 0) |
                           (gate_mode == OMNI_GATE_FULL ? (uintptr_t)(ld_gate * es) : 0);
  const bool aligned = H % 8 == 0 && places % 16 == 0 && (uintptr_t)q % 8 == 0;
  SandwichArgs a{x, residual, post_weight, pre_weight, gate, ldx, ld_residual, ld_gate, ld_residual_out, H, gate_mode,
                 post_eps, pre_eps, residual_scale, residual_out, y, q, scale};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype * 2 + (aligned ? 1 : 0)) {
    case OMNI_DT_BF16 * 2 + 1: return launch_sandwich<OMNI_DT_BF16, true>(a, rows, st);
    case OMNI_DT_BF16 * 2: return launch_sandwich<OMNI_DT_BF16, false>(a, rows, st);
    case OMNI_DT_F16 * 2 + 1: return launch_sandwich<OMNI_DT_F16, true>(a, rows, st);
    case OMNI_DT_F16 * 2: return launch_sandwich<OMNI_DT_F16, false>(a, rows, st);
    case OMNI_DT_F32 * 2 + 1: return launch_sandwich<OMNI_DT_F32, true>(a, rows, st);
    default: return launch_sandwich<OMNI_DT_F32, false>(a, rows, st);
  }
}
