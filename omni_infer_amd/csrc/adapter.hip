// Low-rank adapters of many requests beside a shared projection.
//
//   out[t, :] = base[t, :] + (scale[g] * (x[t, :] . A_g^T)) . B_g^T,     g = the adapter of token t
//
// A_g [S*r, H] holds the S slices of a stacked projection (gate and up), B_g [N, r] their output rows one slice under
// the other; columns of slice j take the columns [j*r, (j+1)*r) of the first product.  The tokens come sorted by
// adapter (sorted_src and offsets of omni_moe_permute with one assignment per token); tokens without an adapter
// follow behind the last group and get their base row.
//
// v = x . A^T is kept in fp32.  The second product wants 16-bit operands on the matrix cores, so v goes in as two of them,
// hi + lo: 16 bits of mantissa in bf16 (off by at most 2^-16 of it), 22 in fp16, where a row is first brought to a largest
// magnitude in [1, 2) by a power of two, since fp16 has no exponents for what 16-bit inputs can add up to.  That costs a
// second matrix instruction, of which there are few: all of this is bound by memory.
//
// Either both products run in one launch, in which every block makes the rows of v it needs, or there are two: the first
// writes v, one row of S*r values per sorted token, the reduction over H cut into `ksplit` parts whose sums lie apart in
// the workspace; the second adds the parts up in order.
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
  int unit_blocks, units;  // column blocks of NB a block of the second product takes, such units over all slices
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

// Row blocks of `bm` rows dealt to the XCDs in runs: work-groups with consecutive numbers go to the 8 XCDs in turn, and an
// XCD that sees a few adapters only keeps their A and B in its L2.  `id` counts the row blocks of a launch, 8 x any number.
__device__ __forceinline__ bool find_tile(const AdapterArgs& g, int none, int bm, int id, RowBlock& rb) {
  const RowBlockScan s = row_blocks_scan(g.offsets, g.n, none, bm);
  const int per = (s.total + 7) / 8, j = id / 8;
  return j < per && row_blocks_find(s, g.offsets, g.n, none, bm, id % 8 * per + j, rb);
}

// ---------------------------------------------------------------- first product
// Operands of 64 consecutive elements of the reduction: lane l of a wavefront holds row l%16 and the elements 8*(l/16)..+7
// of either half, so four lanes read 64 consecutive bytes of a row.
template <int MS, int RT>
struct ShrinkOps {
  v4i x[MS][2], a[RT][2];
};
template <int MS, int RT>
__device__ __forceinline__ void shrink_load(ShrinkOps<MS, RT>& o, const uint16_t* const* xp, const uint16_t* const* ap, int k,
                                            int H, int q) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = min(k + h * 32 + q * 8, H - 8);  // H is a multiple of 8
#pragma unroll
    for (int j = 0; j < RT; ++j) o.a[j][h] = *(const v4i*)(ap[j] + at);
#pragma unroll
    for (int i = 0; i < MS; ++i) o.x[i][h] = *(const v4i*)(xp[i] + at);
  }
}
// what lies past the end of the row or of this wavefront's share counts as zero, in both operands: neither may be finite
template <int MS, int RT>
__device__ __forceinline__ void shrink_cut(ShrinkOps<MS, RT>& o, int k, int k_end, int q) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool in = k + h * 32 + q * 8 < k_end;
#pragma unroll
    for (int j = 0; j < RT; ++j) o.a[j][h] = in ? o.a[j][h] : v4i{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < MS; ++i) o.x[i][h] = in ? o.x[i][h] : v4i{0, 0, 0, 0};
  }
}
template <int DT, int MS, int RT>
__device__ __forceinline__ void shrink_mac(const ShrinkOps<MS, RT>& o, v4f (*acc)[RT]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < MS; ++i)
#pragma unroll
      for (int j = 0; j < RT; ++j) acc[i][j] = mfma_16x16x32<DT>(o.x[i][h], o.a[j][h], acc[i][j]);
}
// The chunks [c0, c_end) of 64 elements, D of them requested at a time.  Nothing that is loaded is carried around the
// loop: the compiler would wait for it there; other wavefronts of the compute unit cover the wait instead.
template <int DT, int MS, int RT, int D>
__device__ __forceinline__ void shrink_chunks(const uint16_t* const* xp, const uint16_t* const* ap, int H, int q, int c0, int c_end,
                                              v4f (*acc)[RT]) {
  const int k_end = min(c_end * KC, H);
#pragma unroll 1
  for (int k = c0 * KC; k < k_end; k += D * KC) {
    ShrinkOps<MS, RT> o[D];
#pragma unroll
    for (int d = 0; d < D; ++d) shrink_load<MS, RT>(o[d], xp, ap, k + d * KC, H, q);
    if (k + D * KC > k_end) {
#pragma unroll
      for (int d = 0; d < D; ++d) shrink_cut<MS, RT>(o[d], k + d * KC, k_end, q);
    }
#pragma unroll
    for (int d = 0; d < D; ++d) shrink_mac<DT, MS, RT>(o[d], acc);
  }
}
__device__ __forceinline__ constexpr int shrink_depth(int MS, int RT) { return MS + RT <= 3 ? 4 : MS + RT <= 5 ? 2 : 1; }

// v = x . A^T for many rows: 128 sorted rows of one adapter by 16*RT of its rows and one part of the reduction.  What bounds
// it is what a compute unit can draw (27 to 30 GB/s), and A counts there like x, so the eight wavefronts share A: chunks of 64
// elements go from memory into LDS, 8 rows of a whole cache line an instruction, two stages in turn, two blocks on a
// compute unit.  Slot s of row r holds piece s ^ ((r>>1)&7) of the row's eight (applied on the global side): the operand
// reads of 16 rows then fall on different banks.  Wavefronts lie 4 (32 rows each) x 2 (half of the A rows each).
#define OMNI_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))
constexpr int ST_ROWS = 128, ST_WAVES = 8;
template <int RT>
struct TileSrc {
  const uint16_t *x[2], *a[RT / 4];  // rows this lane loads, from its piece on
  int px[2], pa[RT / 4];             // its piece's first element
};
template <int RT>
__device__ __forceinline__ void tile_issue(const TileSrc<RT>& t, int k, int H, int w, v4i* __restrict__ dx, v4i* __restrict__ da) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only needs the launch stub
#pragma unroll
  for (int i = 0; i < 2; ++i)
    __builtin_amdgcn_global_load_lds(t.x[i] + min(k + t.px[i], H - 8), OMNI_LDS_PTR(dx + (w * 2 + i) * WAVE), 16, 0, 0);
#pragma unroll
  for (int i = 0; i < RT / 4; ++i)
    __builtin_amdgcn_global_load_lds(t.a[i] + min(k + t.pa[i], H - 8), OMNI_LDS_PTR(da + (w * (RT / 4) + i) * WAVE), 16, 0, 0);
#endif
}
// all loads of this wavefront into LDS have landed, all its reads are done; then the same holds for the block
__device__ __forceinline__ void tile_wait() {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
}
template <int DT, int RT>
__device__ __forceinline__ void tile_mac(const v4i* __restrict__ sx, const v4i* __restrict__ sa, int k, int H, int wr, int wc, int m,
                                         int q, v4f (*acc)[RT / 2]) {
  const int swz = (m >> 1) & 7;  // rows differ by multiples of 16: the same for all of them
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int slot = (h * 4 + q) ^ swz;
    v4i x[2], a[RT / 2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = sx[(wr * 32 + i * 16 + m) * 8 + slot];
#pragma unroll
    for (int j = 0; j < RT / 2; ++j) a[j] = sa[(wc * RT * 8 + j * 16 + m) * 8 + slot];
    if (k + KC > H) {  // past the end of the rows counts as zero, in both operands: neither may be finite
      const bool in = k + h * 32 + q * 8 < H;
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = in ? x[i] : v4i{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < RT / 2; ++j) a[j] = in ? a[j] : v4i{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < RT / 2; ++j) acc[i][j] = mfma_16x16x32<DT>(x[i], a[j], acc[i][j]);
  }
}
template <int DT, int RT>
__global__ __launch_bounds__(ST_WAVES * WAVE, 4) void adapter_shrink_tile_kernel(AdapterArgs g) {
  // separate objects, handed on as __restrict__: a read of one stage does not wait for the loads into the other
  __shared__ __align__(16) v4i sx0[ST_ROWS * 8], sx1[ST_ROWS * 8], sa0[RT * 16 * 8], sa1[RT * 16 * 8];
  RowBlock rb;
  if (!find_tile(g, 0, ST_ROWS, blockIdx.x, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4, wr = w & 3, wc = w >> 2;
  const int c0 = blockIdx.z * RT * 16;
  TileSrc<RT> t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (w * 2 + i) * 8 + lane / 8;
    t.px[i] = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
    t.x[i] = g.x + (size_t)g.sorted_src[rb.row0 + min(row, rb.nrows - 1)] * g.ldx;
  }
#pragma unroll
  for (int i = 0; i < RT / 4; ++i) {
    const int row = (w * (RT / 4) + i) * 8 + lane / 8;
    t.pa[i] = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
    t.a[i] = g.a + ((size_t)rb.group * g.R + min(c0 + row, g.R - 1)) * g.H;
  }
  v4f acc[2][RT / 2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < RT / 2; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  const int chunks = (g.H + KC - 1) / KC, per = (chunks + g.ksplit - 1) / g.ksplit;
  const int c_end = min(chunks, (int)(blockIdx.y + 1) * per);
  int c = blockIdx.y * per;
  if (c < c_end) tile_issue<RT>(t, c * KC, g.H, w, sx0, sa0);
  for (; c < c_end; c += 2) {
    tile_wait();
    if (c + 1 < c_end) tile_issue<RT>(t, (c + 1) * KC, g.H, w, sx1, sa1);
    tile_mac<DT, RT>(sx0, sa0, c * KC, g.H, wr, wc, m, q, acc);
    if (c + 1 >= c_end) break;
    tile_wait();
    if (c + 2 < c_end) tile_issue<RT>(t, (c + 2) * KC, g.H, w, sx0, sa0);
    tile_mac<DT, RT>(sx1, sa1, (c + 1) * KC, g.H, wr, wc, m, q, acc);
  }
  float* vp = g.v + (size_t)blockIdx.y * g.T * g.R;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = wr * 32 + i * 16 + q * 4 + e;
      if (row >= rb.nrows) continue;
#pragma unroll
      for (int j = 0; j < RT / 2; ++j) {
        const int col = c0 + wc * RT * 8 + j * 16 + m;
        if (col < g.R) vp[(size_t)(rb.row0 + row) * g.R + col] = acc[i][j][e];
      }
    }
}

// v = x . A^T.  A block of four wavefronts takes 16*MS sorted rows of one adapter, 16*RT of its rows and one part of
// the reduction, of which every wavefront has its share.
template <int DT, int MS, int RT>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(AdapterArgs g) {
  __shared__ float part[4][16][RT * 16 + 1];
  RowBlock rb;
  if (!find_tile(g, 0, 16 * MS, blockIdx.x, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.z * RT * 16;
  const uint16_t* xp[MS];
#pragma unroll
  for (int i = 0; i < MS; ++i)
    xp[i] = g.x + (size_t)g.sorted_src[rb.row0 + min(i * 16 + m, rb.nrows - 1)] * g.ldx;
  const uint16_t* ap[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j)
    ap[j] = g.a + ((size_t)rb.group * g.R + min(c0 + j * 16 + m, g.R - 1)) * g.H;
  v4f acc[MS][RT];
#pragma unroll
  for (int i = 0; i < MS; ++i)
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  const int chunks = (g.H + KC - 1) / KC;
  const int per = (chunks + g.ksplit * 4 - 1) / (g.ksplit * 4), c_first = (blockIdx.y * 4 + w) * per;
  shrink_chunks<DT, MS, RT, shrink_depth(MS, RT)>(xp, ap, g.H, q, c_first, min(chunks, c_first + per), acc);
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

// ---------------------------------------------------------------- second product
// A value as two 16-bit ones whose sum it is; an infinity or NaN stays in the first
template <int DT>
__device__ __forceinline__ void split16(float f, uint16_t& hi, uint16_t& lo) {
  hi = to_elem<DT>(f);
  const float h = Elem<DT>::cvt(hi);
  lo = fabsf(h) < __builtin_inff() ? to_elem<DT>(f - h) : (uint16_t)0;
}

// 2^-e and 2^e for 2^e <= mx < 2^(e+1), kept within what fp32 holds of both
__device__ __forceinline__ void row_power(float mx, float& down, float& up) {
  const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255) - 127, -100), 100);
  down = __uint_as_float((uint32_t)(127 - e) << 23);
  up = __uint_as_float((uint32_t)(127 + e) << 23);
}

// What one wavefront needs for 64 columns of 16*MS rows: the base values and the first 32*NK of B's reduction.
// Tokens are the columns of the matrix product and output channels its rows, dealt so that a lane ends up with 16
// channels of token l%16 in two runs of 8 (row 4*q + i of tile t is channel 32*(t/2) + 8*q + 4*(t%2) + i).  Moved like that
// an instruction would touch half a cache line of 16 rows, which copies at three quarters of the rate of whole lines (64
// columns of 8192 rows of 4096: 35.6 against 28.0 us); so base and out are moved as whole lines of 8 rows, lane (m, q) with
// row m%8 (+ 8) and run m/8, and the sums change places with lane m^8.
// Ranks up to 16 need one matrix instruction of 32: hi in the first half of the reduction, lo in the second.
template <int MS, int NK>
struct ExpandOps {
  v4i base[MS][2], b[NK][4];  // base[i][h]: row 16*i + 8*h + m%8, columns 32*(m/8) + 8*q ..+7
};
struct Columns {
  const uint16_t* b;  // B of the adapter, first row of the slice
  int width, col0, blk, blk_end;
};
__device__ __forceinline__ const uint16_t* b_row(const AdapterArgs& g, const Columns& c, int blk, int t, int m) {
  return c.b + min(blk * NB + (t >> 1) * 32 + (m >> 2) * 8 + (t & 1) * 4 + (m & 3), c.width - 1) * g.r;
}
// the first of a lane's eight elements of B's reduction
__device__ __forceinline__ int b_col(const AdapterArgs& g, int k, int q) { return min(g.r <= 16 ? (q & 1) * 8 : k + q * 8, g.r - 8); }
// No load is conditional (a condition makes the compiler wait for it on the spot): what is past the last row or column
// repeats the last one and is not stored.
template <int MS, int NK>
__device__ __forceinline__ void expand_load(ExpandOps<MS, NK>& o, const AdapterArgs& g, const Columns& c, int blk, const size_t* tok,
                                            int m, int q) {
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int t = 0; t < 4; ++t) o.b[n][t] = *(const v4i*)(b_row(g, c, blk, t, m) + b_col(g, n * 32, q));
  const int col = c.col0 + min(blk * NB + (m >> 3) * 32 + q * 8, c.width - 8);
#pragma unroll
  for (int i = 0; i < MS; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) o.base[i][h] = *(const v4i*)(g.base + tok[i * 2 + h] * g.ldb + col);
}
// B past the rank counts as zero: v is zero there, but what was loaded in its place need not be finite
__device__ __forceinline__ void b_cut(v4i* b, bool in) {
#pragma unroll
  for (int t = 0; t < 4; ++t) b[t] = in ? b[t] : v4i{0, 0, 0, 0};
}
// the value of lane l^8 (a rotation by 8 inside a row of 16 lanes)
__device__ __forceinline__ float lane_xor8(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
}
template <int DT, int MS>
__device__ __forceinline__ void expand_mac(v4i* b, bool in, const uint16_t* hi, const uint16_t* lo, int at, int step, v4f (*acc)[4]) {
  b_cut(b, in);
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    const v4i vh = *(const v4i*)(hi + at + i * step), vl = *(const v4i*)(lo + at + i * step);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      acc[i][t] = mfma_16x16x32<DT>(b[t], vh, acc[i][t]);
      acc[i][t] = mfma_16x16x32<DT>(b[t], vl, acc[i][t]);
    }
  }
}
template <int DT, int MS, int NK>
__device__ __forceinline__ void expand_block(ExpandOps<MS, NK>& o, const AdapterArgs& g, const Columns& c, int blk,
                                             const RowBlock& rb, bool has, const size_t* tok, int m, int q, const uint16_t* hi,
                                             const uint16_t* lo, int ldk, const float* unscale) {
  v4f acc[MS][4];
#pragma unroll
  for (int i = 0; i < MS; ++i)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[i][t] = v4f{0, 0, 0, 0};
  if (has) {
    if (NK == 1 && g.r <= 16) {
      b_cut(o.b[0], (q & 1) * 8 < g.r);
      const uint16_t* src = ((q >> 1) ? lo : hi) + (q & 1) * 8;
#pragma unroll
      for (int i = 0; i < MS; ++i) {
        const v4i vv = *(const v4i*)(src + (i * 16 + m) * ldk);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = mfma_16x16x32<DT>(o.b[0][t], vv, acc[i][t]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NK; ++n)
        expand_mac<DT, MS>(o.b[n], n * 32 + q * 8 < g.r, hi, lo, m * ldk + n * 32 + q * 8, 16 * ldk, acc);
      if constexpr (NK > 1) {
        for (int k = NK * 32; k < g.r; k += 32) {
          v4i b[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) b[t] = *(const v4i*)(b_row(g, c, blk, t, m) + b_col(g, k, q));
          expand_mac<DT, MS>(b, k + q * 8 < g.r, hi, lo, m * ldk + k + q * 8, 16 * ldk, acc);
        }
      }
    }
  }
  const int col = blk * NB + (m >> 3) * 32 + q * 8;  // this lane's run
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    float un = 1.0f;
    if constexpr (DT == OMNI_DT_F16) un = has ? unscale[i * 16 + m] : 1.0f;
    // runs 0 and 1 of token m become run m/8 of the tokens m%8 and m%8 + 8
    float d[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float r0 = acc[i][e / 4][e % 4] * un, r1 = acc[i][2 + e / 4][e % 4] * un;
      const float other = lane_xor8(m < 8 ? r1 : r0);
      d[0][e] = m < 8 ? r0 : other;
      d[1][e] = m < 8 ? other : r1;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (i * 16 + h * 8 + (m & 7) >= rb.nrows || col >= c.width) continue;  // every lane took part in the exchange
      v4i v = o.base[i][h];
      if (has) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t u = (uint32_t)o.base[i][h][p];
          const float v0 = Elem<DT>::cvt((uint16_t)(u & 0xffffu)) + d[h][2 * p];
          const float v1 = Elem<DT>::cvt((uint16_t)(u >> 16)) + d[h][2 * p + 1];
          if constexpr (DT == OMNI_DT_BF16) v[p] = (int)f32x2_to_bf16x2(v0, v1);
          else v[p] = (int)((uint32_t)to_elem<DT>(v0) | ((uint32_t)to_elem<DT>(v1) << 16));
        }
      }
      *(v4i*)(g.out + tok[i * 2 + h] * g.ldo + c.col0 + col) = v;
    }
  }
}
// which slice and which of its column blocks unit `u` of a launch names; a unit is g.unit_blocks column blocks
__device__ __forceinline__ Columns find_columns(const AdapterArgs& g, int u, int group, int& slice) {
  slice = 0;
  for (; slice < g.slices - 1; ++slice) {
    const int units = ((g.width[slice] + NB - 1) / NB + g.unit_blocks - 1) / g.unit_blocks;
    if (u < units) break;
    u -= units;
  }
  Columns c;
  c.width = g.width[slice];
  c.col0 = g.col0[slice];
  c.b = g.b + ((size_t)min(group, g.n - 1) * g.N + c.col0) * g.r;  // read, not used, by rows without an adapter
  c.blk = u * g.unit_blocks;
  c.blk_end = min((c.width + NB - 1) / NB, c.blk + g.unit_blocks);
  return c;
}

// out = base + v . B^T from the sums of the first launch.  A block of four wavefronts takes 16*MS sorted rows and a
// unit of column blocks; a wavefront takes 64 columns at a time.
template <int DT, int MS, int KQ, int NK>  // ranks up to 64 * KQ, and up to 32 where NK is 1
__global__ __launch_bounds__(256, 4) void adapter_expand_kernel(AdapterArgs g) {
  extern __shared__ __align__(16) uint16_t lds[];  // [2][16*MS][kp + 8]: hi and lo of v, kp = r rounded up to 32 (16)
  __shared__ float unscale[16 * MS];
  RowBlock rb;
  const int none = g.in_place ? 0 : g.T - g.offsets[g.n];
  if (!find_tile(g, none, 16 * MS, blockIdx.x, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const bool has = rb.group < g.n;
  int slice;
  const Columns c = find_columns(g, blockIdx.y, rb.group, slice);
  size_t tok[MS * 2];
#pragma unroll
  for (int i = 0; i < MS * 2; ++i) tok[i] = (size_t)g.sorted_src[rb.row0 + min(i * 8 + (m & 7), rb.nrows - 1)];
  ExpandOps<MS, NK> o;
  int blk = c.blk + w;
  if (blk < c.blk_end) expand_load<MS, NK>(o, g, c, blk, tok, m, q);  // on its way while v is made
  const int kp = g.r <= 16 ? 16 : (g.r + 31) / 32 * 32, ldk = kp + 8;
  uint16_t* hi = lds;
  uint16_t* lo = lds + 16 * MS * ldk;
  if (has) {
    const float sc = g.scale ? g.scale[rb.group] : 1.0f;
    const size_t part = (size_t)g.T * g.R;
    const int l = threadIdx.x % 16;  // a row of v by 16 lanes, four values at a time
#pragma unroll
    for (int i = 0; i < MS; ++i) {
      const int row = i * 16 + threadIdx.x / 16;
      const float* vr = g.v + (size_t)(rb.row0 + min(row, rb.nrows - 1)) * g.R + slice * g.r;
      v4f v[KQ];
      float mx = 0.0f, down = 1.0f;
#pragma unroll
      for (int j = 0; j < KQ; ++j) {
        const int k = (j * 16 + l) * 4;
        const float* p = vr + min(k, g.r - 4);
        v4f s = {0, 0, 0, 0};
        for (int p0 = 0; p0 < g.ksplit; p0 += 4) {
          v4f t[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) t[u] = *(const v4f*)(p + min(p0 + u, g.ksplit - 1) * part);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (p0 + u < g.ksplit) s = s + t[u];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[j][e] = k < g.r ? s[e] * sc : 0.0f;
          if (fabsf(v[j][e]) < __builtin_inff()) mx = fmaxf(mx, fabsf(v[j][e]));
        }
      }
      if constexpr (DT == OMNI_DT_F16) {
        float up;
        row_power(row16_allmax_f(mx), down, up);
        if (l == 0) unscale[row] = up;
      }
#pragma unroll
      for (int j = 0; j < KQ; ++j) {
        const int k = (j * 16 + l) * 4;
        if (k < kp) {
#pragma unroll
          for (int e = 0; e < 4; ++e) split16<DT>(v[j][e] * down, hi[row * ldk + k + e], lo[row * ldk + k + e]);
        }
      }
    }
    __syncthreads();
  }
  if (blk < c.blk_end) expand_block<DT, MS, NK>(o, g, c, blk, rb, has, tok, m, q, hi, lo, ldk, unscale);
  for (blk += 4; blk < c.blk_end; blk += 4) {
    expand_load<MS, NK>(o, g, c, blk, tok, m, q);
    expand_block<DT, MS, NK>(o, g, c, blk, rb, has, tok, m, q, hi, lo, ldk, unscale);
  }
}

// ---------------------------------------------------------------- both products in one launch
// Eight wavefronts, 16 sorted rows of one adapter and a unit of columns of one slice.  The first product is made anew by
// every block of a row block (its operands come from the L2), which saves the launch between the two and the way of v
// through memory.  The blocks of a row block have numbers 8 apart: they run on one XCD and share its L2.
constexpr int FUSED_WAVES = 8;
template <int DT, int RT>
__global__ __launch_bounds__(FUSED_WAVES * WAVE, RT == 1 ? 4 : RT == 2 ? 3 : 2) void adapter_fused_kernel(AdapterArgs g) {
  constexpr int KP = RT * 16 < 32 ? RT * 16 : (RT * 16 + 31) / 32 * 32, LDK = KP + 8;
  __shared__ float part[FUSED_WAVES][16][RT * 16 + 1];
  __shared__ __align__(16) uint16_t lds[2 * 16 * LDK];
  __shared__ float unscale[16];
  const int none = g.in_place ? 0 : g.T - g.offsets[g.n];
  const int unit = (int)blockIdx.x / 8 % g.units;
  RowBlock rb;
  if (!find_tile(g, none, 16, (int)blockIdx.x / 8 / g.units * 8 + (int)blockIdx.x % 8, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const bool has = rb.group < g.n;
  int slice;
  const Columns c = find_columns(g, unit, rb.group, slice);
  const size_t tok[2] = {(size_t)g.sorted_src[rb.row0 + min(m & 7, rb.nrows - 1)],
                         (size_t)g.sorted_src[rb.row0 + min(8 + (m & 7), rb.nrows - 1)]};
  constexpr int NK = RT > 2 ? 2 : 1;
  ExpandOps<1, NK> o;
  int blk = c.blk + w;
  if (blk < c.blk_end) expand_load<1, NK>(o, g, c, blk, tok, m, q);  // on its way during the first product
  if (has) {
    const float sc = g.scale ? g.scale[rb.group] : 1.0f;
    const uint16_t* xp[1] = {g.x + (m < 8 ? tok[0] : tok[1]) * g.ldx};
    const uint16_t* ap[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j)
      ap[j] = g.a + ((size_t)rb.group * g.R + slice * g.r + min(j * 16 + m, g.r - 1)) * g.H;
    v4f acc[1][RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[0][j] = v4f{0, 0, 0, 0};
    const int chunks = (g.H + KC - 1) / KC, per = (chunks + FUSED_WAVES - 1) / FUSED_WAVES;
    shrink_chunks<DT, 1, RT, shrink_depth(1, RT)>(xp, ap, g.H, q, w * per, min(chunks, (w + 1) * per), acc);
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[w][q * 4 + e][j * 16 + m] = acc[0][j][e];
    __syncthreads();
    if (threadIdx.x < 256) {  // a row by 16 lanes
      const int row = threadIdx.x / 16, l = threadIdx.x % 16;
      float v[KP / 16], mx = 0.0f, down = 1.0f;
#pragma unroll
      for (int j = 0; j < KP / 16; ++j) {
        v[j] = 0.0f;
        if (j < RT && j * 16 + l < g.r) {
          float s = part[0][row][j * 16 + l];
#pragma unroll
          for (int p = 1; p < FUSED_WAVES; ++p) s = s + part[p][row][j * 16 + l];
          v[j] = s * sc;
          if (fabsf(v[j]) < __builtin_inff()) mx = fmaxf(mx, fabsf(v[j]));
        }
      }
      if constexpr (DT == OMNI_DT_F16) {
        float up;
        row_power(row16_allmax_f(mx), down, up);
        if (l == 0) unscale[row] = up;
      }
#pragma unroll
      for (int j = 0; j < KP / 16; ++j)
        split16<DT>(v[j] * down, lds[row * LDK + j * 16 + l], lds[(16 + row) * LDK + j * 16 + l]);
    }
    __syncthreads();
  }
  if (blk < c.blk_end) expand_block<DT, 1, NK>(o, g, c, blk, rb, has, tok, m, q, lds, lds + 16 * LDK, LDK, unscale);
  for (blk += FUSED_WAVES; blk < c.blk_end; blk += FUSED_WAVES) {
    expand_load<1, NK>(o, g, c, blk, tok, m, q);
    expand_block<DT, 1, NK>(o, g, c, blk, rb, has, tok, m, q, lds, lds + 16 * LDK, LDK, unscale);
  }
}

int column_units(const AdapterArgs& g, int unit_blocks) {
  int units = 0;
  for (int j = 0; j < g.slices; ++j) units += ((g.width[j] + NB - 1) / NB + unit_blocks - 1) / unit_blocks;
  return units;
}

template <int DT>
int launch_adapter(AdapterArgs& g, const omni_host::AdapterPlan& p, hipStream_t st) {
  g.unit_blocks = p.unit_blocks;
  g.units = column_units(g, p.unit_blocks);
  if (p.fused) {
    const dim3 grid((unsigned)((p.tiles_max + (g.in_place ? 0 : 1) + 7) / 8 * 8 * g.units)), block(FUSED_WAVES * WAVE);
    if (g.r <= 16) hipLaunchKernelGGL((adapter_fused_kernel<DT, 1>), grid, block, 0, st, g);
    else if (g.r <= 32) hipLaunchKernelGGL((adapter_fused_kernel<DT, 2>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((adapter_fused_kernel<DT, 4>), grid, block, 0, st, g);
    OMNI_CHECK_LAUNCH("adapter_linear");
    return OMNI_OK;
  }
#define SHRINK(MS, RT) hipLaunchKernelGGL((adapter_shrink_kernel<DT, MS, RT>), grid, dim3(256), 0, st, g)
#define SHRINK_RT(MS)                       \
  do {                                      \
    if (p.rank_block == 16) SHRINK(MS, 1);  \
    else if (p.rank_block == 32) SHRINK(MS, 2); \
    else if (p.rank_block == 64) SHRINK(MS, 4); \
    else SHRINK(MS, 8);                     \
  } while (0)
  const dim3 grid((unsigned)((p.tiles_max + 7) / 8 * 8), (unsigned)p.ksplit, (unsigned)((g.R + p.rank_block - 1) / p.rank_block));
  if (p.row_tiles == 1) SHRINK_RT(1);
  else if (p.row_tiles == 4) {
    if (p.rank_block == 16) SHRINK(4, 1);
    else SHRINK(4, 2);
  } else if (p.rank_block == 64) hipLaunchKernelGGL((adapter_shrink_tile_kernel<DT, 4>), grid, dim3(ST_WAVES * WAVE), 0, st, g);
  else hipLaunchKernelGGL((adapter_shrink_tile_kernel<DT, 8>), grid, dim3(ST_WAVES * WAVE), 0, st, g);
#undef SHRINK_RT
#undef SHRINK
  OMNI_CHECK_LAUNCH("adapter_linear");
  const int kp = g.r <= 16 ? 16 : (g.r + 31) / 32 * 32;
  const size_t shm = (size_t)2 * 16 * p.out_row_tiles * (kp + 8) * 2;
  const dim3 grid2((unsigned)((p.out_tiles_max + (g.in_place ? 0 : 1) + 7) / 8 * 8), (unsigned)g.units);
#define EXPAND(MS)                                                                                                   \
  do {                                                                                                           \
    if (g.r <= 32) hipLaunchKernelGGL((adapter_expand_kernel<DT, MS, 1, 1>), grid2, dim3(256), shm, st, g);      \
    else if (g.r <= 64) hipLaunchKernelGGL((adapter_expand_kernel<DT, MS, 1, 2>), grid2, dim3(256), shm, st, g); \
    else hipLaunchKernelGGL((adapter_expand_kernel<DT, MS, 4, 2>), grid2, dim3(256), shm, st, g);                \
  } while (0)
  if (p.out_row_tiles == 1) EXPAND(1);
  else EXPAND(2);
#undef EXPAND
  OMNI_CHECK_LAUNCH("adapter_linear");
  return OMNI_OK;
}

}  // namespace

extern "C" size_t omni_adapter_linear_workspace_bytes(int T, int n, int H, int r, int n_slices, int N) {
  if (T <= 0 || n <= 0 || H <= 0 || r <= 0 || n_slices <= 0 || N <= 0) return 0;
  const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, n_slices, N);
  if (p.fused) return 0;
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
  const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, n_slices, (int)N);
  const size_t need = omni_adapter_linear_workspace_bytes(T, n, H, r, n_slices, (int)N);
  if (need && (ws_bytes < need || !workspace)) OMNI_FAIL(OMNI_E_WORKSPACE, "adapter_linear: workspace %zu < %zu", workspace ? ws_bytes : 0, need);
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
  return dtype == OMNI_DT_BF16 ? launch_adapter<OMNI_DT_BF16>(g, p, st) : launch_adapter<OMNI_DT_F16>(g, p, st);
}
