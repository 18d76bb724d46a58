// SwiGLU of rows that exist in memory (+ dynamic int8 quantisation of the result):
//   h = silu(gate) * up, rounded once to the type;  scale = max|h| / 127, q = rint(h / scale) on h as its type holds it
// with gate the first and up the second half of a row, silu(g) = g / (1 + exp(-g)).
// Bound by memory: 3 elements of traffic (and a byte) for about 25 operations.  A block per row; the result stays in
// registers between the row's absmax and its quantisation.
#include "rows.h"

namespace {

struct SwigluArgs {
  const void* gate_up;
  int64_t ld;
  int I;
  void* h;
  int8_t* q;
  float* scale;
};

// The stated exponential ends at exp(87): below -80 the same value comes from two factors, which underflow where the
// quotient does.  -infinity gives NaN, as the quotient of two infinities does.
__device__ __forceinline__ float silu_any(float g) {
  if (g >= -80.0f || g != g) return silu_spec(g);
  if (g < -200.0f) return g * 0.0f;
  const float e = exp_spec(g * 0.5f);
  return (g * e) * e;
}

template <int DT, int THREADS, int MAXV, bool ALIGNED>
__global__ __launch_bounds__(THREADS) void swiglu_quant_kernel(SwigluArgs a) {
  typedef typename Elem<DT>::T ET;
  __shared__ uint32_t redm[THREADS / WAVE];
  const int64_t r = blockIdx.x;
  const int I = a.I, nvec = (I + 7) / 8;
  const ET* gr = (const ET*)a.gate_up + r * a.ld;
  float s[MAXV][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int vi = threadIdx.x + i * THREADS;
    if (vi < nvec) {
      float u[8];
      load8<DT, ALIGNED>(gr, vi, I, s[i]);
      load8<DT, ALIGNED>(gr + I, vi, I, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] = round_to<DT>(silu_any(s[i][j]) * u[j]);
        m = max(m, abs_bits(s[i][j]));
      }
      if (a.h) store8<DT, ALIGNED>((ET*)a.h + r * I, vi, I, s[i]);
    }
  }
  if (a.q == nullptr) return;
  const float sc = block_absmax<THREADS>(m, redm) / 127.0f;
  if (threadIdx.x == 0) a.scale[r] = sc;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int vi = threadIdx.x + i * THREADS;
    if (vi < nvec) store_q8<ALIGNED>(a.q + r * I, vi, I, s[i], sc);
  }
}

constexpr int SWIGLU_MAX_I = 32768;

// Few rows (up to two per compute unit) of more than 2048: 1024 threads with a vector each, 6.2 us for 64 rows of 8192 with
// the int8 output where 256 threads with four each take 9.4.  Many rows: 256 threads, 100 us for 8192 rows of 8192
// (470 MB, 4.7 TB/s) against 103 (512) and 110 us (1024).
template <int DT, bool ALIGNED>
int launch_swiglu(const SwigluArgs& a, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)rows);
#define SWIGLU(THREADS, MAXV) hipLaunchKernelGGL((swiglu_quant_kernel<DT, THREADS, MAXV, ALIGNED>), grid, dim3(THREADS), 0, st, a)
  if (a.I <= 8 * 256) SWIGLU(256, 1);
  else if (a.I > 8 * 1024) SWIGLU(1024, 4);
  else if (rows <= 512) SWIGLU(1024, 1);
  else SWIGLU(256, 4);
#undef SWIGLU
  OMNI_CHECK_LAUNCH("swiglu_quant");
  return OMNI_OK;
}

}  // namespace

extern "C" int omni_swiglu_quant(const void* gate_up, int dtype, int64_t ld, int64_t rows, int I, void* h, int8_t* q,
                                 float* scale, void* stream) {
  if (dtype != OMNI_DT_BF16 && dtype != OMNI_DT_F16 && dtype != OMNI_DT_F32)
    OMNI_FAIL(OMNI_E_INVALID, "swiglu_quant: unknown dtype %d", dtype);
  if (rows < 0 || I <= 0 || ld < 2 * (int64_t)I)
    OMNI_FAIL(OMNI_E_INVALID, "swiglu_quant: bad shape rows=%lld I=%d ld=%lld", (long long)rows, I, (long long)ld);
  if ((q == nullptr) != (scale == nullptr)) OMNI_FAIL(OMNI_E_INVALID, "swiglu_quant: q and scale go together");
  if (rows == 0) return OMNI_OK;
  if (!gate_up) OMNI_FAIL(OMNI_E_INVALID, "swiglu_quant: null pointer");
  if (!h && !q) OMNI_FAIL(OMNI_E_INVALID, "swiglu_quant: no output requested");
  if (I > SWIGLU_MAX_I) OMNI_FAIL(OMNI_E_UNSUPPORTED, "swiglu_quant: I=%d is above %d", I, SWIGLU_MAX_I);
  if (rows > ROWS_MAX) OMNI_FAIL(OMNI_E_UNSUPPORTED, "swiglu_quant: %lld rows, at most %lld", (long long)rows, (long long)ROWS_MAX);
  const size_t es = dtype == OMNI_DT_F32 ? 4 : 2;
  if (((uintptr_t)gate_up | (uintptr_t)h) % es || (uintptr_t)scale % 4) OMNI_FAIL(OMNI_E_INVALID, "swiglu_quant: misaligned pointer");
  const bool aligned = I % 8 == 0 && ((uintptr_t)gate_up | (uintptr_t)h | (uintptr_t)(ld * es)) % 16 == 0 && (uintptr_t)q % 8 == 0;
  SwigluArgs a{gate_up, ld, I, h, q, scale};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype * 2 + (aligned ? 1 : 0)) {
    case OMNI_DT_BF16 * 2 + 1: return launch_swiglu<OMNI_DT_BF16, true>(a, rows, st);
    case OMNI_DT_BF16 * 2: return launch_swiglu<OMNI_DT_BF16, false>(a, rows, st);
    case OMNI_DT_F16 * 2 + 1: return launch_swiglu<OMNI_DT_F16, true>(a, rows, st);
    case OMNI_DT_F16 * 2: return launch_swiglu<OMNI_DT_F16, false>(a, rows, st);
    case OMNI_DT_F32 * 2 + 1: return launch_swiglu<OMNI_DT_F32, true>(a, rows, st);
    default: return launch_swiglu<OMNI_DT_F32, false>(a, rows, st);
  }
}
