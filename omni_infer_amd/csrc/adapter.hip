// Low-rank adapters of many requests beside a shared projection.
//
//   out[t, :] = base[t, :] + (scale[g] * (x[t, :] . A_g^T)) . B_g^T,     g = the adapter of token t
//
// A_g [S*r, H] holds the S slices of a stacked projection (gate and up), B_g [N, r] their output rows one slice under
// the other; columns of slice j take the columns [j*r, (j+1)*r) of the first product.  The tokens come sorted by
// adapter (sorted_src and offsets of omni_moe_permute with one assignment per token); tokens without an adapter
// follow behind the last group and get their base row, and so do those of an adapter whose scale is zero: by the formula a
// row or a matrix that is not finite would turn an adapter that adds nothing into NaN, and base's -0 into 0.
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
constexpr int MAX_WIDTH = 1 << 20, MAX_TOKENS = 1 << 24, MAX_BLOCKS = 1 << 23;  // what indexes and grids hold
constexpr int KC = 64;  // elements of the reduction a wavefront takes at a time: two matrix instructions
constexpr int NB = 64;  // output columns a wavefront takes at a time

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
// Both products take their operands out of LDS.  An operand of the matrix instruction has another row in every lane of 16,
// and loads coalesce over neighbouring lanes only: read like that from memory every lane is an access of its own, and a
// compute unit draws 27 GB/s.  So memory is read 128 bytes of a row by 8 lanes, straight into LDS (lane l of a load writes
// piece l), and the operands are read from there.  Slot s of row r holds piece s ^ ((r>>1)&7) of the row's eight, applied
// on the global side: the 16 rows of an operand read then lie on different banks.
#define OMNI_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))
__device__ __forceinline__ void lds_load16(const uint16_t* src, v4i* dst) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only needs the launch stubs
  __builtin_amdgcn_global_load_lds(src, OMNI_LDS_PTR(dst), 16, 0, 0);
#endif
}
// this wavefront's loads into LDS have landed (and its reads of LDS are done); no access moves across
__device__ __forceinline__ void lds_landed() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  asm volatile("" ::: "memory");
}
// this wavefront's reads of LDS are done: loads may land on what they read
__device__ __forceinline__ void lds_read() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), other counters untouched
  asm volatile("" ::: "memory");
}

// Few rows: 16 rows of x and 16*RT of A in a buffer of the wavefront's own, D chunks of 64 elements at a time.
template <int RT, int D>
struct Stage {
  v4i x[D][16 * 8], a[D][RT * 16 * 8];
};
__device__ __forceinline__ constexpr int shrink_depth(int RT) { return RT <= 1 ? 4 : RT <= 2 ? 2 : 1; }

// acc += the chunks [c0, c_end) of 16 rows of x (lane l: row l%16) by 16*RT rows of A
template <int DT, int RT, int D>
__device__ __forceinline__ void shrink_chunks(Stage<RT, D>& st, const AdapterArgs& g, const RowBlock& rb, const uint16_t* a, int a_rows,
                                              int c0, int c_end, v4f* acc) {
  const int lane = threadIdx.x & (WAVE - 1), m = lane & 15, q = lane >> 4;
  const uint16_t* xp[2];
  int px[2], ao[2 * RT], pa[2 * RT];  // a lane's rows of x and A and the first element of its piece
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = i * 8 + lane / 8;
    xp[i] = g.x + (size_t)g.sorted_src[rb.row0 + min(row, rb.nrows - 1)] * g.ldx;
    px[i] = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
  }
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) {
    const int row = i * 8 + lane / 8;
    ao[i] = min(row, a_rows - 1) * g.H;
    pa[i] = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
  }
  const int k_end = min(c_end * KC, g.H), swz = (m >> 1) & 7;
#pragma unroll 1
  for (int k = c0 * KC; k < k_end; k += D * KC) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int kd = k + d * KC;  // past the end the last elements come again, and count as zero below
#pragma unroll
      for (int i = 0; i < 2 * RT; ++i) lds_load16(a + ao[i] + min(kd + pa[i], g.H - 8), st.a[d] + i * WAVE);
#pragma unroll
      for (int i = 0; i < 2; ++i) lds_load16(xp[i] + min(kd + px[i], g.H - 8), st.x[d] + i * WAVE);
    }
    lds_landed();
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int slot = (h * 4 + q) ^ swz;
        v4i x = st.x[d][m * 8 + slot], av[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) av[j] = st.a[d][(j * 16 + m) * 8 + slot];
        if (k + (d + 1) * KC > k_end) {  // zero in both operands: neither may be finite
          const bool in = k + d * KC + h * 32 + q * 8 < k_end;
          x = in ? x : v4i{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < RT; ++j) av[j] = in ? av[j] : v4i{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j] = mfma_16x16x32<DT>(x, av[j], acc[j]);
      }
    lds_read();
  }
}

// v = x . A^T for many rows: 128 sorted rows of one adapter by 16*RT of its rows and one part of the reduction.  What bounds
// it is what a compute unit can draw from behind its cache, 27 to 30 GB/s whether the L2 has it or not, and A counts there
// like x, so the eight wavefronts share A: chunks of 64 elements go into two stages in turn, two blocks on a compute unit.
// Wavefronts lie 4 (32 rows each) x 2 (half of the A rows each).  8192 x 7168 tokens by 128 rows of A in 35 to 41 us (117 MB
// of x, 3 TB/s), where 64 rows a block with operands straight from memory took 72: the L2 counts 287 MB of requests, 128 MB of
// them hits (A), 27 GB/s for each of 256 compute units.  8192 x 2048 by 16 rows in 12 us.
constexpr int ST_ROWS = 128, ST_WAVES = 8;
template <int RT>
struct TileSrc {
  const uint16_t *x[2], *a[RT / 4];  // rows this lane loads, from its piece on
  int px[2], pa[RT / 4];             // its piece's first element
};
template <int RT>
__device__ __forceinline__ void tile_issue(const TileSrc<RT>& t, int k, int H, int w, v4i* __restrict__ dx, v4i* __restrict__ da) {
#pragma unroll
  for (int i = 0; i < 2; ++i) lds_load16(t.x[i] + min(k + t.px[i], H - 8), dx + (w * 2 + i) * WAVE);
#pragma unroll
  for (int i = 0; i < RT / 4; ++i) lds_load16(t.a[i] + min(k + t.pa[i], H - 8), da + (w * (RT / 4) + i) * WAVE);
}
// all loads of this wavefront into LDS have landed, all its reads are done; then the same holds for the block
__device__ __forceinline__ void tile_wait() {
  lds_landed();
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

// v = x . A^T for few rows.  A block of four wavefronts takes 16 sorted rows of one adapter, 16*RT of its rows and one part of
// the reduction, of which every wavefront has its share.  A single token waits for memory (rank 32 and 64, 7168 -> 2 x 2048:
// 3.2 and 5.3 us in 14 parts, with 5.3 and 6.0 us for the second product); an adapter per token is bound by A: 64 tokens, about 56
// adapters in use, rank 32 and 64: 51 and 103 MB in 11 and 22 us, 4.6 TB/s.
template <int DT, int RT>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(AdapterArgs g) {
  constexpr int D = shrink_depth(RT);
  union Shared {
    Stage<RT, D> stage[4];
    float part[4][16][RT * 16 + 1];
  };
  __shared__ __align__(16) Shared sh;
  RowBlock rb;
  if (!find_tile(g, 0, 16, blockIdx.x, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.z * RT * 16;
  v4f acc[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j] = v4f{0, 0, 0, 0};
  const int chunks = (g.H + KC - 1) / KC;
  const int per = (chunks + g.ksplit * 4 - 1) / (g.ksplit * 4), c_first = (blockIdx.y * 4 + w) * per;
  shrink_chunks<DT, RT, D>(sh.stage[w], g, rb, g.a + ((size_t)rb.group * g.R + c0) * g.H, g.R - c0, c_first,
                           min(chunks, c_first + per), acc);
  __syncthreads();  // the stages are done with
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) sh.part[w][q * 4 + e][j * 16 + m] = acc[j][e];
  __syncthreads();
  float* vp = g.v + (size_t)blockIdx.y * g.T * g.R;
  for (int t = threadIdx.x; t < 16 * RT * 16; t += 256) {
    const int row = t / (RT * 16), c = t % (RT * 16);
    if (row < rb.nrows && c0 + c < g.R)
      vp[(size_t)(rb.row0 + row) * g.R + c0 + c] =
          ((sh.part[0][row][c] + sh.part[1][row][c]) + sh.part[2][row][c]) + sh.part[3][row][c];
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

// A wavefront takes 64 columns of 16*MS rows at a time.  Tokens are the rows of the matrix product and output channels its
// columns, dealt so that lane (m, q) ends up with the four channels 4*m..+3 (tile t: channel 4*m + t) of the tokens
// 16*i + 4*q + e: 16 neighbouring lanes move a whole cache line of base and of out.
// Ranks up to 16 need one matrix instruction of 32: hi in the first half of the reduction, lo in the second.
struct Columns {
  const uint16_t* b;  // B of the adapter, first row of the slice
  int width, col0, blk, blk_end;
};
template <int MS>
struct ExpandOps {
  v2i base[MS][4];
};
// B of 64 channels and up to 64 of the rank (8*P elements a row), in a buffer of the wavefront's own: 64 rows of P pieces of 16
// bytes one after the other, the piece at place p with the low three bits of its number changed by higher ones, so that
// the reads of rows 4*m + t fall on different banks.
__device__ __forceinline__ int panel_place(int unit) {
  const int x = unit >> 3;
  return unit ^ ((x ^ (x >> 1) ^ (x >> 2)) & 7);
}
template <int PMAX>
struct Panel {
  int row_piece[PMAX];  // what this lane loads: row | piece << 8
};
template <int PMAX>
__device__ __forceinline__ void panel_setup(Panel<PMAX>& pn, int P) {
  const int lane = threadIdx.x & (WAVE - 1);
#pragma unroll
  for (int i = 0; i < PMAX; ++i) {
    const int unit = panel_place(i * WAVE + lane);
    pn.row_piece[i] = unit / P | (unit % P) << 8;
  }
}
template <int PMAX>
__device__ __forceinline__ void panel_issue(const Panel<PMAX>& pn, int P, const AdapterArgs& g, const Columns& c, int blk, int kc,
                                            v4i* panel) {
#pragma unroll
  for (int i = 0; i < PMAX; ++i) {
    if (i >= P) break;
    const int row = min(blk * NB + (pn.row_piece[i] & 255), c.width - 1), k = min(kc + (pn.row_piece[i] >> 8) * 8, g.r - 8);
    lds_load16(c.b + row * g.r + k, panel + i * WAVE);
  }
}
// No load is conditional (a condition makes the compiler wait for it on the spot): what is past the last row or column
// repeats the last one and is not stored.
// `tok` holds the tokens of the rows in LDS: read anew for every block, so that no addresses of rows are kept in registers.
template <int MS>
__device__ __forceinline__ void base_load(ExpandOps<MS>& o, const AdapterArgs& g, const Columns& c, int blk, const v4i* tok, int m,
                                          int q) {
  const int col = c.col0 + min(blk * NB + m * 4, c.width - 4);
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    const v4i t = tok[i * 4 + q];
#pragma unroll
    for (int e = 0; e < 4; ++e) o.base[i][e] = *(const v2i*)(g.base + (size_t)t[e] * g.ldb + col);
  }
}
// one column block whose panel (the first 64 of the rank) and base values are here or on their way
template <int DT, int MS, int PMAX>
__device__ __forceinline__ void expand_block(const ExpandOps<MS>& o, const Panel<PMAX>& pn, int P, v4i* panel, const AdapterArgs& g,
                                             const Columns& c, int blk, const RowBlock& rb, bool has, float sc, const v4i* tok,
                                             int m, int q, const uint16_t* hi, const uint16_t* lo, int ldk, const float* unscale) {
  v4f acc[MS][4];
#pragma unroll
  for (int i = 0; i < MS; ++i)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[i][t] = v4f{0, 0, 0, 0};
  if (has) {
    lds_landed();
    if (g.r <= 16) {
      const int k = (q & 1) * 8;
      const uint16_t* src = ((q >> 1) ? lo : hi) + k;
      v4i b[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        b[t] = panel[panel_place((m * 4 + t) * P + min(q & 1, P - 1))];
        b[t] = k < g.r ? b[t] : v4i{0, 0, 0, 0};  // v is zero there, but what stands in B's place need not be finite
      }
#pragma unroll
      for (int i = 0; i < MS; ++i) {
        const v4i v = *(const v4i*)(src + (i * 16 + m) * ldk);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = mfma_16x16x32<DT>(v, b[t], acc[i][t]);
      }
    } else {
      for (int kc = 0;;) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int k = kc + n * 32;
          if (k >= g.r) break;
          v4i b[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            b[t] = panel[panel_place((m * 4 + t) * P + min(n * 4 + q, P - 1))];
            b[t] = k + q * 8 < g.r ? b[t] : v4i{0, 0, 0, 0};
          }
#pragma unroll
          for (int i = 0; i < MS; ++i) {
            const int at = (i * 16 + m) * ldk + k + q * 8;
            const v4i vh = *(const v4i*)(hi + at), vl = *(const v4i*)(lo + at);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              acc[i][t] = mfma_16x16x32<DT>(vh, b[t], acc[i][t]);
              acc[i][t] = mfma_16x16x32<DT>(vl, b[t], acc[i][t]);
            }
          }
        }
        kc += 64;
        if (kc >= g.r) break;
        lds_read();
        panel_issue<PMAX>(pn, P, g, c, blk, kc, panel);
        lds_landed();
      }
    }
  }
  const int col = blk * NB + m * 4;
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    asm volatile("" ::: "memory");
    const v4i t = tok[i * 4 + q];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = i * 16 + q * 4 + e;
      if (row >= rb.nrows || col >= c.width) continue;
      v2i v = o.base[i][e];
      if (sc != 0.0f) {
        float un = 1.0f;
        if constexpr (DT == OMNI_DT_F16) un = unscale[row];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint32_t u = (uint32_t)o.base[i][e][p];
          const float v0 = Elem<DT>::cvt((uint16_t)(u & 0xffffu)) + acc[i][2 * p][e] * un;
          const float v1 = Elem<DT>::cvt((uint16_t)(u >> 16)) + acc[i][2 * p + 1][e] * un;
          if constexpr (DT == OMNI_DT_BF16) v[p] = (int)f32x2_to_bf16x2(v0, v1);
          else v[p] = (int)((uint32_t)to_elem<DT>(v0) | ((uint32_t)to_elem<DT>(v1) << 16));
        }
      }
      *(v2i*)(g.out + (size_t)t[e] * g.ldo + c.col0 + col) = v;
    }
  }
}
// The column blocks of one wavefront.  The first block's panel and base values are on their way when `o` and `blk` come in.
template <int DT, int MS, int PMAX>
__device__ __forceinline__ void expand_columns(ExpandOps<MS>& o, const Panel<PMAX>& pn, int P, v4i* panel, const AdapterArgs& g,
                                               const Columns& c, int blk, int step, const RowBlock& rb, bool has, float sc, const v4i* tok,
                                               int m, int q, const uint16_t* hi, const uint16_t* lo, int ldk, const float* unscale) {
  for (bool first = true; blk < c.blk_end; blk += step, first = false) {
    if (!first) {
      if (has) {
        lds_read();
        panel_issue<PMAX>(pn, P, g, c, blk, 0, panel);
      }
      base_load<MS>(o, g, c, blk, tok, m, q);
    }
    expand_block<DT, MS, PMAX>(o, pn, P, panel, g, c, blk, rb, has, sc, tok, m, q, hi, lo, ldk, unscale);
  }
}
// the tokens of a block's rows; rows past the last repeat it
template <int MS>
__device__ __forceinline__ void load_tokens(const AdapterArgs& g, const RowBlock& rb, v4i* tok) {
  if (threadIdx.x < 16 * MS) ((int*)tok)[threadIdx.x] = g.sorted_src[rb.row0 + min((int)threadIdx.x, rb.nrows - 1)];
  __syncthreads();
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

// the parts of a sum in order, U of them requested at a time
template <int U>
__device__ __forceinline__ v4f sum_parts(const float* p, size_t step, int n) {
  v4f s = {0, 0, 0, 0};
  for (int p0 = 0; p0 < n; p0 += U) {
    v4f t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = *(const v4f*)(p + min(p0 + u, n - 1) * step);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p0 + u < n) s = s + t[u];
  }
  return s;
}
// out = base + v . B^T from the sums of the first launch.  A block of four wavefronts takes 16*MS sorted rows and a
// unit of column blocks; a wavefront takes 64 columns at a time.  Bound by base and out, which a plain copy moves in 26 us for
// 8192 rows of 2 x 2048 and in 45 to 49 us for 8192 of 7168: 51 us at rank 64 (MS = 2; B and the parts of v, read by every
// block, are more again: 379 MB of requests to the L2, 210 MB of them hits, 30 GB/s for each compute unit) and 55 us at rank 16
// (MS = 1: more wavefronts; MS = 2 takes 61).  16 column blocks a unit: 32 take 56 and 62 us.
template <int DT, int MS, int KQ, int PMAX>  // ranks up to 64 * KQ and, below 64, up to 8 * PMAX
__global__ __launch_bounds__(256, MS == 2 ? 3 : PMAX == 4 ? 5 : 4) void adapter_expand_kernel(AdapterArgs g) {
  // [4][64 * P] pieces of B, then [2][16*MS][kp + 8]: hi and lo of v, kp = r rounded up to 32 (16)
  extern __shared__ __align__(16) v4i dyn[];
  __shared__ __align__(16) v4i tok[4 * MS];
  __shared__ float unscale[16 * MS];
  RowBlock rb;
  const int none = g.in_place ? 0 : g.T - g.offsets[g.n];
  const int unit = (int)blockIdx.x / 8 % g.units;  // the units of a row block run one after the other on one XCD
  if (!find_tile(g, none, 16 * MS, (int)blockIdx.x / 8 / g.units * 8 + (int)blockIdx.x % 8, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const bool has = rb.group < g.n;
  float sc = 0.0f;  // of a group without an adapter, too: nothing is added
  int slice;
  const Columns c = find_columns(g, unit, rb.group, slice);
  const int P = min(g.r, 64) / 8;
  v4i* panel = dyn + w * WAVE * P;
  Panel<PMAX> pn;
  panel_setup<PMAX>(pn, P);
  load_tokens<MS>(g, rb, tok);
  ExpandOps<MS> o;
  const int blk = c.blk + w;
  if (blk < c.blk_end) {  // on its way while v is made
    if (has) panel_issue<PMAX>(pn, P, g, c, blk, 0, panel);
    base_load<MS>(o, g, c, blk, tok, m, q);
  }
  const int kp = g.r <= 16 ? 16 : (g.r + 31) / 32 * 32, ldk = kp + 8;
  uint16_t* hi = (uint16_t*)(dyn + 4 * WAVE * P);
  uint16_t* lo = hi + 16 * MS * ldk;
  if (has) {
    sc = g.scale ? g.scale[rb.group] : 1.0f;
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
        const v4f s = g.ksplit > 4 ? sum_parts<8>(p, part, g.ksplit) : sum_parts<4>(p, part, g.ksplit);
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
  expand_columns<DT, MS, PMAX>(o, pn, P, panel, g, c, blk, 4, rb, has, sc, tok, m, q, hi, lo, ldk, unscale);
}

// ---------------------------------------------------------------- both products in one launch
// Eight wavefronts, 16 sorted rows of one adapter and a unit of columns of one slice.  The first product is made anew by
// every block of a row block (its operands come from the L2), which saves the launch between the two and the way of v
// through memory.  The blocks of a row block have numbers 8 apart: they run on one XCD and share its L2.
// Bound by latency: the launch and, at H = 7168 and rank 16, six trips to memory in a row (offsets, tokens, and a wavefront's 14
// chunks four at a time).  One token, rank 16, 7168 -> 2 x 2048: 8.5 us.  64 tokens, each with an adapter of its own (some 56 of 64; the
// others have none), rank 16, 2048 -> 7168: 11 us for 19 MB.
constexpr int FUSED_WAVES = 8;
template <int DT, int RT>
__global__ __launch_bounds__(FUSED_WAVES * WAVE) void adapter_fused_kernel(AdapterArgs g) {
  constexpr int KP = RT * 16 < 32 ? RT * 16 : (RT * 16 + 31) / 32 * 32, LDK = KP + 8, D = shrink_depth(RT), PMAX = 2 * RT;
  union Shared {
    Stage<RT, D> stage[FUSED_WAVES];
    float part[FUSED_WAVES][16][RT * 16 + 1];
  };
  __shared__ __align__(16) Shared sh;
  __shared__ __align__(16) v4i panels[FUSED_WAVES][WAVE * PMAX];
  __shared__ __align__(16) uint16_t lds[2 * 16 * LDK];
  __shared__ __align__(16) v4i tok[4];
  __shared__ float unscale[16];
  const int none = g.in_place ? 0 : g.T - g.offsets[g.n];
  const int unit = (int)blockIdx.x / 8 % g.units;
  RowBlock rb;
  if (!find_tile(g, none, 16, (int)blockIdx.x / 8 / g.units * 8 + (int)blockIdx.x % 8, rb)) return;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  const int m = lane & 15, q = lane >> 4;
  const bool has = rb.group < g.n;
  float sc = 0.0f;  // of a group without an adapter, too: nothing is added
  int slice;
  const Columns c = find_columns(g, unit, rb.group, slice);
  const int P = g.r / 8;
  v4i* panel = panels[w];
  Panel<PMAX> pn;
  panel_setup<PMAX>(pn, P);
  load_tokens<1>(g, rb, tok);
  ExpandOps<1> o;
  const int blk = c.blk + w;
  if (blk < c.blk_end) {  // on its way during the first product
    if (has) panel_issue<PMAX>(pn, P, g, c, blk, 0, panel);
    base_load<1>(o, g, c, blk, tok, m, q);
  }
  if (has) {
    sc = g.scale ? g.scale[rb.group] : 1.0f;
    v4f acc[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = v4f{0, 0, 0, 0};
    const int chunks = (g.H + KC - 1) / KC, per = (chunks + FUSED_WAVES - 1) / FUSED_WAVES;
    shrink_chunks<DT, RT, D>(sh.stage[w], g, rb, g.a + ((size_t)rb.group * g.R + slice * g.r) * g.H, g.r, w * per,
                             min(chunks, (w + 1) * per), acc);
    __syncthreads();  // the stages are done with
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sh.part[w][q * 4 + e][j * 16 + m] = acc[j][e];
    __syncthreads();
    if (threadIdx.x < 256) {  // a row by 16 lanes
      const int row = threadIdx.x / 16, l = threadIdx.x % 16;
      float v[KP / 16], mx = 0.0f, down = 1.0f;
#pragma unroll
      for (int j = 0; j < KP / 16; ++j) {
        v[j] = 0.0f;
        if (j < RT && j * 16 + l < g.r) {
          float s = sh.part[0][row][j * 16 + l];
#pragma unroll
          for (int p = 1; p < FUSED_WAVES; ++p) s = s + sh.part[p][row][j * 16 + l];
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
  expand_columns<DT, 1, PMAX>(o, pn, P, panel, g, c, blk, FUSED_WAVES, rb, has, sc, tok, m, q, lds, lds + 16 * LDK, LDK, unscale);
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
#define SHRINK(RT) hipLaunchKernelGGL((adapter_shrink_kernel<DT, RT>), grid, dim3(256), 0, st, g)
#define SHRINK_TILE(RT) hipLaunchKernelGGL((adapter_shrink_tile_kernel<DT, RT>), grid, dim3(ST_WAVES * WAVE), 0, st, g)
  const dim3 grid((unsigned)((p.tiles_max + 7) / 8 * 8), (unsigned)p.ksplit, (unsigned)((g.R + p.rank_block - 1) / p.rank_block));
  if (p.row_tiles == 8) {
    if (p.rank_block == 64) SHRINK_TILE(4);
    else SHRINK_TILE(8);
  } else {
    if (p.rank_block == 16) SHRINK(1);
    else if (p.rank_block == 32) SHRINK(2);
    else if (p.rank_block == 64) SHRINK(4);
    else SHRINK(8);
  }
#undef SHRINK_TILE
#undef SHRINK
  OMNI_CHECK_LAUNCH("adapter_linear");
  const int kp = g.r <= 16 ? 16 : (g.r + 31) / 32 * 32;
  const size_t shm = (size_t)4 * WAVE * (g.r < 64 ? g.r / 8 : 8) * 16 + (size_t)2 * 16 * p.out_row_tiles * (kp + 8) * 2;
  const dim3 grid2((unsigned)((p.out_tiles_max + (g.in_place ? 0 : 1) + 7) / 8 * 8 * g.units));
#define EXPAND(MS, KQ, PMAX) hipLaunchKernelGGL((adapter_expand_kernel<DT, MS, KQ, PMAX>), grid2, dim3(256), shm, st, g)
  if (p.out_row_tiles == 2) {  // ranks of 33 to 128
    if (g.r <= 64) EXPAND(2, 1, 8);
    else EXPAND(2, 4, 8);
  } else {
    if (g.r <= 32) EXPAND(1, 1, 4);
    else if (g.r <= 64) EXPAND(1, 1, 8);
    else EXPAND(1, 4, 8);
  }
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
  if (((int64_t)p.out_tiles_max + 8) * (N / 64 / p.unit_blocks + n_slices) > MAX_BLOCKS)
    OMNI_FAIL(OMNI_E_UNSUPPORTED, "adapter_linear: %d tokens of %lld columns", T, (long long)N);
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
