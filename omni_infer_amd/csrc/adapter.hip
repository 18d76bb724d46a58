// Low-rank adapters of many requests beside a shared projection.
//
//   out[t, :] = base[t, :] + (scale[g] * (x[t, :] . A_g^T)) . B_g^T,     g = the adapter of token t
//
// A_g [S*r, H] holds the S slices of a stacked projection (gate and up), B_g [N, r] their output rows one slice under
// the other; columns of slice j take the columns [j*r, (j+1)*r) of the first product.  The tokens come sorted by
// adapter (sorted_src and offsets of omni_moe_permute with one assignment per token); tokens without an adapter
// follow behind the last group and get their base row.
//
// Two launches.  The first makes v = x . A^T, one row of S*r values per sorted token, the reduction over H cut into
// `ksplit` parts whose sums lie apart in the workspace; the second adds the parts up in order, scales, multiplies
// with B and adds the base.  v is kept in fp32.  The second product wants 16-bit operands on the matrix cores, so v
// goes in as two of them, hi + lo: 16 bits of mantissa in bf16 (off by at most 2^-16 of it), 22 in fp16, where a row is first
// brought to a largest magnitude in [1, 2) by a power of two, since fp16 has no exponents for what 16-bit inputs can
// add up to.  That costs a second matrix instruction, of which there are few: both launches are bound by memory.
#include "rows.h"

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int MAX_SLICES = 4;
constexpr int MAX_RANK = 256;
constexpr int MAX_ADAPTERS = 256;
constexpr int MAX_WIDTH = 1 << 20, MAX_TOKENS = 1 << 24;  // what the grids hold
constexpr int KC = 64;        // elements of the reduction a wavefront takes at a time: two matrix instructions
constexpr int NB = 64;        // output columns a wavefront takes at a time

struct AdapterArgs {
  const uint16_t *x, *base, *a, *b;
  const float* scale;
  const int32_t *sorted_src, *offsets;
  int64_t ldx, ldb, ldo;
  int T, n, H, r, R, N, slices;
  int width[MAX_SLICES], col0[MAX_SLICES];
  int ksplit;
  int in_place;
  int blocks_per_slice_chunk;  // column blocks of NB a block of the second launch takes
  uint16_t* out;
  float* v;  // [ksplit][T][R]
};

template <int DT>
__device__ __forceinline__ v4f mfma_16x16x32(v4i a, v4i b, v4f c) {
  if constexpr (DT == OMNI_DT_BF16) {
    v8bf x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  } else {
    v8h x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  }
}

// v = x . A^T.  A block of four wavefronts takes 16*MS sorted rows of one adapter, 16*RT of its rows and one part of
// the reduction; the wavefronts share the part, 64 elements in turn.  Lane l of a wavefront holds row l%16 and the
// elements 16*(l/16)..+15 of the 64: both operands use the same order, so the sum is the same and four lanes read a
// whole cache line.
template <int DT, int MS, int RT>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(AdapterArgs g) {
  __shared__ float part[4][16][RT * 16 + 1];
  RowBlock rb;
  if (!find_row_block(g.offsets, g.n, 0, 16 * MS, blockIdx.x, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.z * RT * 16;
  const uint16_t* xp[MS];
#pragma unroll
  for (int i = 0; i < MS; ++i)
    xp[i] = g.x + (size_t)g.sorted_src[rb.row0 + min(i * 16 + m, rb.nrows - 1)] * g.ldx + q * 16;
  const uint16_t* ap[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j)
    ap[j] = g.a + ((size_t)rb.group * g.R + min(c0 + j * 16 + m, g.R - 1)) * g.H + q * 16;
  v4f acc[MS][RT];
#pragma unroll
  for (int i = 0; i < MS; ++i)
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  const int chunks = (g.H + KC - 1) / KC;
  const int per = (chunks + g.ksplit - 1) / g.ksplit;
  const int c_end = min(chunks, (int)(blockIdx.y + 1) * per);
  for (int c = blockIdx.y * per + w; c < c_end; c += 4) {
    const int k = c * KC;
    // H is a multiple of 8: each half of a lane's 16 elements is inside or outside as a whole
    const bool in0 = k + q * 16 < g.H, in1 = k + q * 16 + 8 < g.H;
    v4i xv[MS][2], av[RT][2];
#pragma unroll
    for (int i = 0; i < MS; ++i) {
      xv[i][0] = in0 ? *(const v4i*)(xp[i] + k) : v4i{0, 0, 0, 0};
      xv[i][1] = in1 ? *(const v4i*)(xp[i] + k + 8) : v4i{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      av[j][0] = in0 ? *(const v4i*)(ap[j] + k) : v4i{0, 0, 0, 0};
      av[j][1] = in1 ? *(const v4i*)(ap[j] + k + 8) : v4i{0, 0, 0, 0};
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MS; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[i][j] = mfma_16x16x32<DT>(xv[i][h], av[j][h], acc[i][j]);
  }
  float* vp = g.v + (size_t)blockIdx.y * g.T * g.R;
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    if (i) __syncthreads();  // the sums of the rows before have been read
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[w][q * 4 + e][j * 16 + m] = acc[i][j][e];
    __syncthreads();
    for (int t = threadIdx.x; t < 16 * RT * 16; t += 256) {
      const int row = t / (RT * 16), c = t % (RT * 16);
      if (i * 16 + row < rb.nrows && c0 + c < g.R)
        vp[(size_t)(rb.row0 + i * 16 + row) * g.R + c0 + c] =
            ((part[0][row][c] + part[1][row][c]) + part[2][row][c]) + part[3][row][c];
    }
  }
}

// A value as two 16-bit ones whose sum it is; an infinity or NaN stays in the first
template <int DT>
__device__ __forceinline__ void split16(float f, uint16_t& hi, uint16_t& lo) {
  hi = to_elem<DT>(f);
  const float h = Elem<DT>::cvt(hi);
  lo = fabsf(h) < __builtin_inff() ? to_elem<DT>(f - h) : (uint16_t)0;
}

// out = base + v . B^T.  A block of four wavefronts takes 16*MS sorted rows and some column blocks of one slice; a
// wavefront takes 64 columns at a time.  Tokens are the columns of the matrix product and output channels its rows,
// dealt so that a lane ends up with 16 consecutive channels of one token (row 4*q + i of tile t is channel
// 16*q + 4*t + i): base and out move as whole cache lines.
// Ranks up to 16 need one matrix instruction of 32: hi in the first half of the reduction, lo in the second.
template <int DT, int MS>
__global__ __launch_bounds__(256) void adapter_expand_kernel(AdapterArgs g) {
  extern __shared__ __align__(16) uint16_t lds[];  // [2][16*MS][kp + 8]: hi and lo of v, kp = r rounded up to 32 (16)
  __shared__ float unscale[16 * MS];
  RowBlock rb;
  const int none = g.in_place ? 0 : g.T - g.offsets[g.n];
  if (!find_row_block(g.offsets, g.n, none, 16 * MS, blockIdx.x, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  // which slice and which of its column blocks
  int slice = 0, blk0 = blockIdx.y * g.blocks_per_slice_chunk;
  for (; slice < g.slices - 1; ++slice) {
    const int cols = (g.width[slice] + NB - 1) / NB;
    const int chunks = (cols + g.blocks_per_slice_chunk - 1) / g.blocks_per_slice_chunk;
    if (blk0 < chunks * g.blocks_per_slice_chunk) break;
    blk0 -= chunks * g.blocks_per_slice_chunk;
  }
  const int width = g.width[slice], col0 = g.col0[slice];
  const int blk_end = min((width + NB - 1) / NB, blk0 + g.blocks_per_slice_chunk);
  const bool packed = g.r <= 16;
  const int kp = packed ? 16 : (g.r + 31) / 32 * 32, ldk = kp + 8;
  const bool has = rb.group < g.n;
  uint16_t* hi = lds;
  uint16_t* lo = lds + 16 * MS * ldk;
  if (has) {
    const float sc = g.scale ? g.scale[rb.group] : 1.0f;
    // a row of v by 16 lanes
    for (int row = threadIdx.x / 16; row < 16 * MS; row += 16) {
      const float* vr = g.v + (size_t)(rb.row0 + min(row, rb.nrows - 1)) * g.R + slice * g.r;
      float up = 1.0f;
      if constexpr (DT == OMNI_DT_F16) {
        float mx = 0.0f;
        for (int c = m; c < g.r; c += 16) {
          float s = 0.0f;
          for (int p = 0; p < g.ksplit; ++p) s = s + vr[(size_t)p * g.T * g.R + c];
          s = fabsf(s * sc);
          if (s < __builtin_inff()) mx = fmaxf(mx, s);
        }
        mx = row16_allmax_f(mx);
        // 2^-e for 2^e <= mx < 2^(e+1), within what fp32 holds of both factors
        const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255) - 127, -100), 100);
        up = __uint_as_float((uint32_t)(127 - e) << 23);
        if (m == 0) unscale[row] = __uint_as_float((uint32_t)(127 + e) << 23);
      }
      for (int c = m; c < kp; c += 16) {
        float s = 0.0f;
        if (c < g.r) {
          for (int p = 0; p < g.ksplit; ++p) s = s + vr[(size_t)p * g.T * g.R + c];
          s = (s * sc) * up;
        }
        split16<DT>(s, hi[row * ldk + c], lo[row * ldk + c]);
      }
    }
    __syncthreads();
  }
  size_t tok[MS];
#pragma unroll
  for (int i = 0; i < MS; ++i) tok[i] = (size_t)g.sorted_src[rb.row0 + min(i * 16 + m, rb.nrows - 1)];
  const uint16_t* bp = g.b + ((size_t)rb.group * g.N + col0) * g.r;
  for (int blk = blk0 + w; blk < blk_end; blk += 4) {
    const int n0 = blk * NB;
    const int nl = n0 + q * 16;  // this lane's first channel
    v4i bv[MS][2];
#pragma unroll
    for (int i = 0; i < MS; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (i * 16 + m < rb.nrows && nl + h * 8 < width)
          bv[i][h] = __builtin_nontemporal_load((const v4i*)(g.base + tok[i] * g.ldb + col0 + nl + h * 8));
    v4f acc[MS][4];
#pragma unroll
    for (int i = 0; i < MS; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[i][t] = v4f{0, 0, 0, 0};
    if (has) {
      const uint16_t* brow[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) brow[t] = bp + (size_t)min(n0 + (m >> 2) * 16 + t * 4 + (m & 3), width - 1) * g.r;
      if (packed) {
        const int k8 = (q & 1) * 8;
        v4i av[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) av[t] = k8 < g.r ? *(const v4i*)(brow[t] + k8) : v4i{0, 0, 0, 0};
        const uint16_t* src = (q >> 1) ? lo : hi;
#pragma unroll
        for (int i = 0; i < MS; ++i) {
          const v4i vv = *(const v4i*)(src + (i * 16 + m) * ldk + k8);
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[i][t] = mfma_16x16x32<DT>(av[t], vv, acc[i][t]);
        }
      } else {
        for (int k = q * 8; k < kp; k += 32) {
          v4i av[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) av[t] = k < g.r ? *(const v4i*)(brow[t] + k) : v4i{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < MS; ++i) {
            const v4i vh = *(const v4i*)(hi + (i * 16 + m) * ldk + k), vl = *(const v4i*)(lo + (i * 16 + m) * ldk + k);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              acc[i][t] = mfma_16x16x32<DT>(av[t], vh, acc[i][t]);
              acc[i][t] = mfma_16x16x32<DT>(av[t], vl, acc[i][t]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MS; ++i) {
      if (i * 16 + m >= rb.nrows) continue;
      float un = 1.0f;
      if constexpr (DT == OMNI_DT_F16) un = has ? unscale[i * 16 + m] : 1.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (nl + h * 8 >= width) continue;
        v4i o = bv[i][h];
        if (has) {
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const v4f& d = acc[i][h * 2 + p / 2];
            const uint32_t u = (uint32_t)bv[i][h][p];
            const float lo16 = Elem<DT>::cvt((uint16_t)(u & 0xffffu)) + d[(p & 1) * 2] * un;
            const float hi16 = Elem<DT>::cvt((uint16_t)(u >> 16)) + d[(p & 1) * 2 + 1] * un;
            o[p] = (int)((uint32_t)to_elem<DT>(lo16) | ((uint32_t)to_elem<DT>(hi16) << 16));
          }
        }
        __builtin_nontemporal_store(o, (v4i*)(g.out + tok[i] * g.ldo + col0 + nl + h * 8));
      }
    }
  }
}

template <int DT, int MS>
int launch_adapter(AdapterArgs& g, const omni_host::AdapterPlan& p, hipStream_t st) {
  if (p.tiles_max > 0) {
    const dim3 grid((unsigned)p.tiles_max, (unsigned)p.ksplit, (unsigned)((g.R + p.rank_block - 1) / p.rank_block));
    if (p.rank_block == 16) hipLaunchKernelGGL((adapter_shrink_kernel<DT, MS, 1>), grid, dim3(256), 0, st, g);
    else if (p.rank_block == 32) hipLaunchKernelGGL((adapter_shrink_kernel<DT, MS, 2>), grid, dim3(256), 0, st, g);
    else if (p.rank_block == 64) hipLaunchKernelGGL((adapter_shrink_kernel<DT, MS, 4>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((adapter_shrink_kernel<DT, MS, 8>), grid, dim3(256), 0, st, g);
    OMNI_CHECK_LAUNCH("adapter_linear");
  }
  g.blocks_per_slice_chunk = p.col_blocks;
  int chunks = 0;
  for (int j = 0; j < g.slices; ++j) chunks += ((g.width[j] + NB - 1) / NB + p.col_blocks - 1) / p.col_blocks;
  const int kp = g.r <= 16 ? 16 : (g.r + 31) / 32 * 32;
  const size_t shm = (size_t)2 * 16 * MS * (kp + 8) * 2;
  hipLaunchKernelGGL((adapter_expand_kernel<DT, MS>), dim3((unsigned)(p.tiles_max + (g.in_place ? 0 : 1)), (unsigned)chunks),
                     dim3(256), shm, st, g);
  OMNI_CHECK_LAUNCH("adapter_linear");
  return OMNI_OK;
}

}  // namespace

extern "C" size_t omni_adapter_linear_workspace_bytes(int T, int n, int H, int r, int n_slices) {
  if (T <= 0 || n <= 0 || H <= 0 || r <= 0 || n_slices <= 0) return 0;
  const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, n_slices);
  return align256((size_t)p.ksplit * T * r * n_slices * sizeof(float));
}

extern "C" int omni_adapter_linear(const void* x, int dtype, int64_t ldx, const void* base, int64_t ld_base, const void* a,
                                   const void* b, const float* scale, const int32_t* sorted_src, const int32_t* offsets,
                                   int T, int n, int H, int r, int n_slices, const int32_t* widths, void* out,
                                   int64_t ld_out, void* workspace, size_t ws_bytes, void* stream) {
  if (dtype != OMNI_DT_BF16 && dtype != OMNI_DT_F16) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: dtype %d is not bf16 or fp16", dtype);
  if (T < 0 || n <= 0 || H <= 0 || r <= 0 || n_slices <= 0)
    OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: bad sizes T=%d n=%d H=%d r=%d slices=%d", T, n, H, r, n_slices);
  if (n_slices > MAX_SLICES) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: %d slices, at most %d", n_slices, MAX_SLICES);
  if (!widths) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: null pointer");
  AdapterArgs g{};
  int64_t N = 0;
  for (int j = 0; j < n_slices; ++j) {
    if (widths[j] <= 0) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: slice %d has %d columns", j, widths[j]);
    if (widths[j] % 8) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: slice %d has %d columns, not a multiple of 8", j, widths[j]);
    g.width[j] = widths[j];
    g.col0[j] = (int)N;
    N += widths[j];
  }
  if (N > MAX_WIDTH) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: %lld columns, at most %d", (long long)N, MAX_WIDTH);
  if (H % 8 || H > MAX_WIDTH) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: H=%d is not a multiple of 8 up to %d", H, MAX_WIDTH);
  if (T > MAX_TOKENS) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: %d tokens, at most %d", T, MAX_TOKENS);
  if (r % 8 || r > MAX_RANK) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: rank %d is not a multiple of 8 up to %d", r, MAX_RANK);
  if (n > MAX_ADAPTERS) OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: %d adapters, at most %d", n, MAX_ADAPTERS);
  if (ldx < H || ld_base < N || ld_out < N) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: a row stride is below the row's length");
  if (T == 0) return OMNI_OK;
  if (!x || !base || !a || !b || !sorted_src || !offsets || !out) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: null pointer");
  if (((uintptr_t)x | (uintptr_t)base | (uintptr_t)a | (uintptr_t)b | (uintptr_t)out) % 16 || ldx % 8 || ld_base % 8 || ld_out % 8 ||
      ((uintptr_t)scale | (uintptr_t)sorted_src | (uintptr_t)offsets) % 4)
    OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: misaligned pointer or row stride");
  if (out == base && ld_out != ld_base) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: out is base with another row stride");
  const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, n_slices);
  const size_t need = omni_adapter_linear_workspace_bytes(T, n, H, r, n_slices);
  if (ws_bytes < need || !workspace) OMNI_FAIL(OMNI_E_WORKSPACE, "adapter_linear: workspace %zu < %zu", workspace ? ws_bytes : 0, need);
  if ((uintptr_t)workspace % 16) OMNI_FAIL(OMNI_E_INVALID, "adapter_linear: misaligned workspace");
  g.x = (const uint16_t*)x;
  g.base = (const uint16_t*)base;
  g.a = (const uint16_t*)a;
  g.b = (const uint16_t*)b;
  g.scale = scale;
  g.sorted_src = sorted_src;
  g.offsets = offsets;
  g.ldx = ldx;
  g.ldb = ld_base;
  g.ldo = ld_out;
  g.T = T;
  g.n = n;
  g.H = H;
  g.r = r;
  g.R = r * n_slices;
  g.N = (int)N;
  g.slices = n_slices;
  g.ksplit = p.ksplit;
  g.in_place = out == base;
  g.out = (uint16_t*)out;
  g.v = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == OMNI_DT_BF16)
    return p.row_tiles == 1 ? launch_adapter<OMNI_DT_BF16, 1>(g, p, st) : launch_adapter<OMNI_DT_BF16, 4>(g, p, st);
  return p.row_tiles == 1 ? launch_adapter<OMNI_DT_F16, 1>(g, p, st) : launch_adapter<OMNI_DT_F16, 4>(g, p, st);
}
