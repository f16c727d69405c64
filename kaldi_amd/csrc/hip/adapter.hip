// Low-rank adapters of many speakers beside one shared affine layer: hipI32_adapter_plan, hipF_adapter_forward,
// hipF_adapter_backward (include/kaldi_hip.h has the formulas).
//
// A float product on this chip's fp32 matrix instructions is bound at 157 TFLOP/s; on bfloat16 they do 2.5 PFLOP/s.
// So every operand is split, where it is loaded, into three bfloat16 numbers that add up to it exactly (8 bits of
// mantissa each, rounded to nearest: |x - hi| <= 2^-9 |x|, |x - hi - mid| <= 2^-18 |x|, the rest fits lo), and a product
// is the sum of the six part products down to 2^-18 of it, accumulated in float by the matrix instruction: the bfloat16x3
// decomposition published by Henry, Tang and Heinecke (2019).  The three products left out are at most
// 2 * 2^-27 + 2^-36 of the product, an eighth of a float's rounding.  An infinity splits into
// inf + NaN; so does, at first, a finite float that rounds to infinity (first_part has what is done about it).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

// ---- eight floats as three fragments of eight bfloat16 ----------------------------------------------------------
struct Frag {
  v8b hi, mid, lo;
};
// Two floats at a time: x - hi comes from the instruction that adds two bfloat16 products to a float, with the factors -1
// and 0 (exact: the difference is a float); unpacking hi first would take two instructions more.  The factors are kept in
// scalar registers: as literals the assembler takes -1 for the upper half only.
struct Minus {
  v2b first, second;
};
__device__ __forceinline__ Minus minus_ones() {
  unsigned f = 0x0000bf80u, s = 0xbf800000u;
  asm("" : "+s"(f), "+s"(s));
  return {__builtin_bit_cast(v2b, f), __builtin_bit_cast(v2b, s)};
}
// The first part.  What rounds to infinity, a finite float beyond the largest finite bfloat16, has a rest of minus infinity and
// one of NaN: every sum that it is in is NaN.  CLAMP takes the largest finite bfloat16 instead, so that the rest is finite (that of
// infinity is infinity, and the rest of that NaN).  It would be one instruction in seven more, 1 to 4 % of every call; so a
// kernel goes over its operands without, and where a sum has come out as NaN, once more with it (2048 -> 2048 with such operands:
// 256 rows 36 to 47 us instead of 30, 4096 rows 320 to 360 instead of 230).
template <bool CLAMP>
__device__ __forceinline__ v2b first_part(float x, float y) {
  constexpr float most = 0x1.fep+127f;
  if (CLAMP) x = __builtin_amdgcn_fmed3f(x, -most, most), y = __builtin_amdgcn_fmed3f(y, -most, most);
  return __builtin_convertvector((v2f){x, y}, v2b);
}
template <bool CLAMP>
__device__ __forceinline__ void split2(float x, float y, v2b &hi, v2b &mid, v2b &lo) {
  const Minus one = minus_ones();
  hi = first_part<CLAMP>(x, y);
  x = __builtin_amdgcn_fdot2_f32_bf16(hi, one.first, x, false);
  y = __builtin_amdgcn_fdot2_f32_bf16(hi, one.second, y, false);
  mid = __builtin_convertvector((v2f){x, y}, v2b);
  x = __builtin_amdgcn_fdot2_f32_bf16(mid, one.first, x, false);
  y = __builtin_amdgcn_fdot2_f32_bf16(mid, one.second, y, false);
  lo = __builtin_convertvector((v2f){x, y}, v2b);
}
// the same with the parts unpacked and subtracted: where the matrix instructions keep the vector unit waiting anyway (the
// tiled kernel), this measures 3 % faster than the above, in the kernels that split more than they multiply 6 % slower
template <bool CLAMP>
__device__ __forceinline__ void split2_apart(float x, float y, v2b &hi, v2b &mid, v2b &lo) {
  hi = first_part<CLAMP>(x, y);
  x -= (float)hi.x, y -= (float)hi.y;
  mid = __builtin_convertvector((v2f){x, y}, v2b);
  x -= (float)mid.x, y -= (float)mid.y;
  lo = __builtin_convertvector((v2f){x, y}, v2b);
}
template <bool CLAMP = true, bool APART = false>
__device__ __forceinline__ Frag split8(const float (&x)[8]) {
  Frag f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    v2b h, m, l;
    if (APART) split2_apart<CLAMP>(x[i], x[i + 1], h, m, l);
    else split2<CLAMP>(x[i], x[i + 1], h, m, l);
    f.hi[i] = h.x, f.hi[i + 1] = h.y;
    f.mid[i] = m.x, f.mid[i + 1] = m.y;
    f.lo[i] = l.x, f.lo[i + 1] = l.y;
  }
  return f;
}
template <int N>
__device__ __forceinline__ bool any_nan(const v4f (&v)[N]) {
  bool nan = false;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) nan |= v[j][i] != v[j][i];
  return nan;
}
// c + small += a * b.  hi * hi has a sum of its own, which is then rounded once per step and not six times: what the matrix
// instruction drops of a sum has a sign more often than not, and a gradient over many rows adds such errors up (8192 rows of
// 2048 -> 2048, 4 adapters of rank 32: 1.6e-7 of the gradient's norm instead of 1.9e-6, at the same speed).
__device__ __forceinline__ void mfma6(const Frag &a, const Frag &b, v4f &c, v4f &small) {
  small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.lo, b.hi, small, 0, 0, 0);
  small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.hi, b.lo, small, 0, 0, 0);
  small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.mid, b.mid, small, 0, 0, 0);
  small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.mid, b.hi, small, 0, 0, 0);
  small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.hi, b.mid, small, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.hi, b.hi, c, 0, 0, 0);
}

// ---- operand loads ------------------------------------------------------------------------------------------------
// The 16x16x32 instruction: lane l holds eight elements of row l % 16 of A and of column l % 16 of B, and gets
// D[4 (l / 16) + i][l % 16], i = 0..3.  Which of a step's 32 inner indices the eight are is free as long as A and B agree:
// with q = l / 16 they are 4 q .. 4 q + 3 and 16 + 4 q .. 16 + 4 q + 3, so that one load of 16 bytes per lane covers whole
// 64-byte pieces of 16 rows.
__device__ __forceinline__ int inner(int q, int e) { return 4 * q + (e & 3) + 4 * (e & 4); }

// the lane's eight of a row at `row` (which points at the step's first), zeros from `left` on
template <bool VEC>
__device__ __forceinline__ void load_row8(const float *row, int q, int left, float (&x)[8]) {
  if (VEC && left >= 32) {
    const v4f a = *reinterpret_cast<const v4f *>(row + 4 * q), b = *reinterpret_cast<const v4f *>(row + 16 + 4 * q);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = inner(q, e) < left ? row[inner(q, e)] : 0.f;
  }
}
// NB neighbouring floats of a row from column c, zeros from C on
template <int NB, bool VEC>
__device__ __forceinline__ void load_cols(const float *row, int c, int C, float (&x)[NB]) {
  if (VEC && NB == 4 && c + 4 <= C) {
    const v4f a = *reinterpret_cast<const v4f *>(row + c);
    x[0] = a.x, x[1 % NB] = a.y, x[2 % NB] = a.z, x[3 % NB] = a.w;
  } else if (VEC && NB == 2 && c + 2 <= C) {
    const v2f a = *reinterpret_cast<const v2f *>(row + c);
    x[0] = a.x, x[1 % NB] = a.y;
  } else {
#pragma unroll
    for (int j = 0; j < NB; ++j) x[j] = c + j < C ? row[c + j] : 0.f;
  }
}

// Rows whose lanes would each ask for another 16 bytes cost one request per lane; eight lanes that ask for 128 bytes of a
// row cost one.  So a wave has the rows of a step copied into its own piece of LDS, eight rows per instruction, and
// takes its operands from there.  Slot 8 r + c (16 bytes) holds the four floats c ^ (r & 7) of row r, so that the eight lanes
// that read the same four of eight rows find them in different banks.
__device__ __forceinline__ void stage_rows(const float *row, int lane, float *to) {  // `row`: of lane / 8, at the step's first
  typedef __attribute__((address_space(1))) const void gvoid;
  typedef __attribute__((address_space(3))) void lvoid;
  __builtin_amdgcn_global_load_lds((gvoid *)(row + 4 * ((lane & 7) ^ (lane >> 3))), (lvoid *)to, 16, 0, 0);
}
__device__ __forceinline__ void staged_row8(const float *piece, int r, int q, float (&x)[8]) {
  const v4f a = *reinterpret_cast<const v4f *>(piece + 32 * r + 4 * (q ^ (r & 7)));
  const v4f b = *reinterpret_cast<const v4f *>(piece + 32 * r + 4 * ((4 + q) ^ (r & 7)));
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void staged_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void staged_taken() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---- which adapter ------------------------------------------------------------------------------------------------
struct Stack {
  int num, max_rank, rows;
  const int32_t *begin;
  const float *scale;
};
// the stack rows of adapter g (0 <= g < num): first row and how many, inside the stack whatever begin[] holds
__device__ __forceinline__ void stack_rows(const Stack &st, int g, int *first, int *rank) {
  int lo = st.begin[g], hi = st.begin[g + 1];
  lo = min(max(lo, 0), st.rows);
  hi = max(min(hi, st.rows), lo);  // (a difference of what lies inside: it cannot wrap around)
  *first = lo;
  *rank = min(hi - lo, st.max_rank);
}

// Row `i` of the tile sequence: the row itself or order[i]; -1 behind the end or outside the matrix.
__device__ __forceinline__ int row_of(const int32_t *order, int i, int N) {
  if (i >= N) return -1;
  if (!order) return i;
  const int r = order[i];
  return (unsigned)r < (unsigned)N ? r : -1;
}
__device__ __forceinline__ int adapter_of(const int32_t *row_adapter, int num, int row) {
  if (row < 0 || num == 0) return -1;
  const int g = row_adapter[row];
  return (unsigned)g < (unsigned)num ? g : -1;
}

// The runs of equal adapters among the (up to 64) rows of a tile, as every lane of a wave sees them: lane m has the
// adapter of tile row m.  `starts` marks the first rows of runs that have an adapter, `changes` the first rows of all.
struct Runs {
  unsigned long long starts, changes;
};
__device__ __forceinline__ Runs find_runs(int g, int lane) {
  const int prev = __shfl_up(g, 1, 64);
  const bool change = lane == 0 || prev != g;
  Runs r;
  r.changes = __ballot(change);
  r.starts = __ballot(change && g >= 0);
  return r;
}
// rows of the run that starts at bit s
__device__ __forceinline__ unsigned long long run_mask(const Runs &r, int s) {
  const unsigned long long above = s == 63 ? 0ull : (r.changes >> (s + 1)) << (s + 1);
  const unsigned long long from = ~0ull << s;
  return above ? from & ((above & (0ull - above)) - 1ull) : from;
}

// ---- grouping of a bunch --------------------------------------------------------------------------------------------
// One workgroup per adapter (and one for the rows without): counts the rows in front of its group, then writes its rows
// in ascending order.  Every workgroup reads all ids (from the L2: N * (num + 1) * 8 bytes in all); no atomics, no
// scratch, a stable order.  Made for bunches: 256 rows of 40 adapters 2 to 5 us, 4096 of 200 6.3, 65536 of 200 63 us, 2^20 of 200
// 1.0 ms, of 2000 5.1 ms.
__global__ __launch_bounds__(1024) void plan_kernel(const int32_t *row_adapter, int N, int num, int32_t *order,
                                                    int32_t *row_begin) {
  __shared__ int part[16];
  const int me = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int before = 0;
  for (int i = threadIdx.x; i < N; i += blockDim.x) {
    const unsigned g = (unsigned)row_adapter[i];
    before += (g < (unsigned)num ? (int)g : num) < me;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
  if (lane == 0) part[wave] = before;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < waves; ++w) at += part[w];
  __syncthreads();
  if (threadIdx.x == 0) row_begin[me] = at;
  for (int i0 = 0; i0 < N; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    bool mine = false;
    if (i < N) {
      const unsigned g = (unsigned)row_adapter[i];
      mine = (g < (unsigned)num ? (int)g : num) == me;
    }
    const unsigned long long hits = __ballot(mine);
    if (lane == 0) part[wave] = __popcll(hits);
    __syncthreads();
    int place = at;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) place += part[w];
      at += part[w];
    }
    if (mine) order[place + __popcll(hits & ((1ull << lane) - 1ull))] = i;
    __syncthreads();
  }
}

// ---- the narrow product: t = s_g * x * side_g^T ----------------------------------------------------------------------
// One workgroup per window of up to 16 rows and block of 16 * NB rank columns; its eight waves take steps of 32 of the
// inner dimension in turn and add up through LDS in a fixed order.  A window of several adapters is gone through
// once per run of equal adapters; only the run's rows are kept from a pass, so nothing of one row reaches another.  Bound
// by reading x (4096 x 2048: 16 us, 2.1 TB/s) or, for few rows, by latency (1 to 64 rows: 6.3 us, with 4, 8 or 16 waves).
struct NarrowArgs {
  const float *x; int ldx, N, K;
  const float *side; int ldside;
  Stack st;
  const int32_t *row_adapter, *order;
  int window;
  float *t; int ldt;
};
constexpr int kNarrowWaves = 8;
template <int NB, bool VEC>
struct NarrowShared {
  float stage[VEC ? kNarrowWaves * (16 + 16 * NB) * 32 : 4];
  float part[kNarrowWaves][16][16 * NB + 4];
  int rows[16];
  float scale[16];
};
// (waves behind the eighth, of a larger workgroup, have nothing to do: the order of the sums is the same in every kernel)
template <int NB, bool VEC>
__device__ __forceinline__ void narrow_block(const NarrowArgs &p, int block_x, int block_y, NarrowShared<NB, VEC> &sh) {
  constexpr int NW = kNarrowWaves;
  const float *x = p.x, *side = p.side;
  const int ldx = p.ldx, N = p.N, K = p.K, lds = p.ldside, window = p.window;
  const Stack &st = p.st;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, q = lane >> 4;
  const int first_row = block_x * window, col0 = block_y * 16 * NB;
  const int32_t *order = window > 1 ? p.order : nullptr;  // (nothing to put together: a load less to wait for, 1.4 us)
  const int row = lane < window ? row_of(order, first_row + lane, N) : -1;
  const int g = adapter_of(p.row_adapter, st.num, row);
  const Runs runs = find_runs(g, lane);
  const int my_row = __shfl(row, l15, 64);
  const float *xr = x + (size_t)max(my_row, 0) * ldx;
  if (wave == 0 && lane < 16) {  // for the end; asked for now
    sh.rows[lane] = row;
    sh.scale[lane] = g >= 0 && st.scale ? st.scale[g] : 1.f;
  }
  v4f total[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) total[j] = (v4f){0.f, 0.f, 0.f, 0.f};
  for (unsigned long long left = wave < NW ? runs.starts : 0ull; left; left &= left - 1ull) {
    const int s = __builtin_ctzll(left);
    const unsigned long long mask = run_mask(runs, s);
    int lo, rank;
    stack_rows(st, __shfl(g, s, 64), &lo, &rank);
    if (rank <= col0) continue;
    const float *br[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) br[j] = side + (size_t)(lo + min(col0 + NB * l15 + j, rank - 1)) * lds;
    v4f acc[NB], small[NB];
    auto sweep = [&](auto clamp) {
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[j] = small[j] = (v4f){0.f, 0.f, 0.f, 0.f};
      int k0 = 32 * wave;
      if (VEC && k0 + 32 <= K) {
        float *piece = sh.stage + wave * (16 + 16 * NB) * 32;
        const float *sx[2], *sb[2 * NB];
#pragma unroll
        for (int i = 0; i < 2; ++i) sx[i] = x + (size_t)max(__shfl(row, 8 * i + (lane >> 3), 64), 0) * ldx;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          const int r = 8 * i + (lane >> 3);  // piece row 16 j + l: the stack's row NB l + j
          sb[i] = side + (size_t)(lo + min(col0 + NB * (r & 15) + (r >> 4), rank - 1)) * lds;
        }
        auto ask = [&](int k) {
#pragma unroll
          for (int i = 0; i < 2; ++i) stage_rows(sx[i] + k, lane, piece + 256 * i);
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) stage_rows(sb[i] + k, lane, piece + 512 + 256 * i);
        };
        ask(k0);
        for (; k0 + 32 <= K; k0 += 32 * NW) {
          float a[8], b[NB][8];
          staged_arrived();
          staged_row8(piece, l15, q, a);
#pragma unroll
          for (int j = 0; j < NB; ++j) staged_row8(piece + 512, 16 * j + l15, q, b[j]);
          staged_taken();
          if (k0 + 32 * NW + 32 <= K) ask(k0 + 32 * NW);
          const Frag fa = split8<clamp.value>(a);
#pragma unroll
          for (int j = 0; j < NB; ++j) mfma6(fa, split8<clamp.value>(b[j]), acc[j], small[j]);
        }
      }
      for (; k0 < K; k0 += 32 * NW) {
        float a[8], b[NB][8];
        load_row8<VEC>(xr + k0, q, K - k0, a);
#pragma unroll
        for (int j = 0; j < NB; ++j) load_row8<VEC>(br[j] + k0, q, K - k0, b[j]);
        const Frag fa = split8<clamp.value>(a);
#pragma unroll
        for (int j = 0; j < NB; ++j) mfma6(fa, split8<clamp.value>(b[j]), acc[j], small[j]);
      }
    };
    sweep(std::false_type());
    if (__ballot(any_nan(small))) sweep(std::true_type());
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((mask >> (4 * q + i)) & 1ull && col0 + NB * l15 + j < rank) total[j][i] = acc[j][i] + small[j][i];
  }
  if (wave < NW) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sh.part[wave][4 * q + i][NB * l15 + j] = total[j][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < window * 16 * NB; e += blockDim.x) {
    const int m = e / (16 * NB), c = e % (16 * NB);
    const int r = sh.rows[m];
    if (r < 0 || col0 + c >= st.max_rank) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += sh.part[w][m][c];
    v *= sh.scale[m];
    p.t[(size_t)r * p.ldt + col0 + c] = v;
  }
}

template <int NB, bool VEC>
__global__ __launch_bounds__(64 * kNarrowWaves) void narrow_kernel(NarrowArgs p) {
  __shared__ __align__(16) NarrowShared<NB, VEC> sh;
  narrow_block<NB, VEC>(p, blockIdx.x, blockIdx.y, sh);
}

// ---- the wide product -----------------------------------------------------------------------
struct WideArgs {
  const float *x; int ldx;       // rows x K
  const float *w; int ldw;       // NN: K x C, else C x K
  int N, K, C;
  const float *bias;             // C or null
  const float *t; int ldt;       // rows x max_rank (null: no adapters)
  const float *side; int ldside; // stack x C
  Stack st;
  const int32_t *row_adapter, *order;
  const float *y; int ldy;       // derivative of the sigmoid below, or null
  int act;
  float *out; int ldout;
  int tiles_m, tiles_n;
};

// One workgroup per tile of 16 * MB rows and 16 * NB columns.  Its NW waves take steps of 32 of the inner dimension in turn
// (no wave needs what another loads, so there is no barrier: a wave waits for its own piece of LDS) and add up through LDS
// in a fixed order.  The columns of a lane are neighbours: block j of the tile holds columns NB * l + j.
// FN > 0: the narrow product (FN: its NB) runs in the same launch, in the workgroups in front; the adapters' part, the
// activation and the derivative below follow in a launch of their own, finish_kernel.  Three launches' chains of dependent
// loads become two: one frame of 2048 -> 2048 10.4 us (narrow, then wide with the adapters' part: 12.9), 64 rows of 1024 ->
// 1483 10.9 (16.1), 256 rows of 2048 -> 2048 with their plan 30.1 (35.0; 1 us more with the narrow product's workgroups behind
// the tiles', 3 with 4 rows in each instead of one).
// 256 rows, 2048 -> 2048 alone (32x64 tiles): 20 us, of which some 13 are splitting and multiplying (9 and 6 at full rate,
// hardly overlapped), 7 start and end; 107 TFLOP/s of float products.  One row: 7.2 us for 16.8 MB of weights, three quarters
// of it the latencies of a kernel of dependent loads.  Loads straight into the registers' layout (16 bytes of another row
// per lane) cap at 9 TB/s from the L2: 33 us for those 256 rows.
template <int MB, int NB, int NW, bool NN, bool VEC, int FN>
__global__ __launch_bounds__(64 * NW) void wide_kernel(WideArgs p, NarrowArgs narrow, int windows, int narrow_blocks) {
  constexpr int BM = 16 * MB, BN = 16 * NB, STAGED = NN ? BM : BM + BN;
  constexpr int SHARED = VEC && STAGED * 32 > BM * BN ? STAGED * 32 : BM * BN;
  using Narrow = NarrowShared<FN ? FN : 1, VEC>;
  constexpr int BYTES = NW * SHARED * 4;
  __shared__ __align__(16) char shared_s[FN && (int)sizeof(Narrow) > BYTES ? (int)sizeof(Narrow) : BYTES];
  if (FN && (int)blockIdx.x < narrow_blocks)
    return narrow_block<FN ? FN : 1, VEC>(narrow, blockIdx.x % windows, blockIdx.x / windows, *reinterpret_cast<Narrow *>(shared_s));
  float *stage_s = reinterpret_cast<float *>(shared_s);  // a wave's rows of a step; at the end its sums
  float (*part)[BM][BN] = reinterpret_cast<float (*)[BM][BN]>(stage_s);
  static_assert(64 * NW % BN == 0, "a thread finishes one column");
  // tiles of the same columns run on one of the 8 dies, so that a piece of W comes into one L2 only
  const int block = blockIdx.x - (FN ? narrow_blocks : 0), die = block & 7, local = block >> 3;
  const int tile_n = die + 8 * (local / p.tiles_m), tile_m = local % p.tiles_m;
  if (tile_n >= p.tiles_n) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, q = lane >> 4;
  const int m0 = tile_m * BM, n0 = tile_n * BN, c0 = n0 + NB * l15;
  const float *xr[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) xr[b] = p.x + (size_t)min(m0 + 16 * b + l15, p.N - 1) * p.ldx;
  v4f acc[MB][NB], small[MB][NB];

  const float *wr[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) wr[j] = p.w + (size_t)min(c0 + j, p.C - 1) * p.ldw;
  struct Step {
    float a[MB][8], b[NB][8];
  };
  auto load = [&](int k0, int left, Step &s) {
#pragma unroll
    for (int m = 0; m < MB; ++m) load_row8<VEC>(xr[m] + k0, q, left, s.a[m]);
    if (NN) {
      const float *w = p.w + (size_t)k0 * p.ldw;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v[NB] = {};
        if (inner(q, e) < left) load_cols<NB, VEC>(w + (size_t)inner(q, e) * p.ldw, c0, p.C, v);
#pragma unroll
        for (int j = 0; j < NB; ++j) s.b[j][e] = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < NB; ++j) load_row8<VEC>(wr[j] + k0, q, left, s.b[j]);
    }
  };
  auto multiply = [&](const Step &s, auto clamp) {
    Frag fa[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) fa[m] = split8<clamp.value>(s.a[m]);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const Frag fb = split8<clamp.value>(s.b[j]);
#pragma unroll
      for (int m = 0; m < MB; ++m) mfma6(fa[m], fb, acc[m][j], small[m][j]);
    }
  };
  const int my_c = n0 + threadIdx.x % BN;
  const float my_bias = p.bias && my_c < p.C ? p.bias[my_c] : 0.f;  // for the end; asked for now
  constexpr int D = 32 * NW;
  auto sweep = [&](auto clamp) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[m][j] = small[m][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    int k0 = 32 * wave;
    if (VEC && k0 + 32 <= p.K) {
      float *piece = stage_s + wave * STAGED * 32;
      const float *sx[2 * MB], *sw[2 * NB];
#pragma unroll
      for (int i = 0; i < 2 * MB; ++i) sx[i] = p.x + (size_t)min(m0 + 8 * i + (lane >> 3), p.N - 1) * p.ldx;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const int r = 8 * i + (lane >> 3);  // piece row 16 j + l: row NB l + j of the tile's part of W
        sw[i] = p.w + (size_t)min(n0 + NB * (r & 15) + (r >> 4), p.C - 1) * p.ldw;
      }
      float raw[8][NB];  // (NN: rows of W along the tile's columns, straight into registers)
      auto ask = [&](int k) {
#pragma unroll
        for (int i = 0; i < 2 * MB; ++i) stage_rows(sx[i] + k, lane, piece + 256 * i);
        if (NN) {
          const float *w = p.w + (size_t)k * p.ldw;
#pragma unroll
          for (int e = 0; e < 8; ++e) load_cols<NB, VEC>(w + (size_t)inner(q, e) * p.ldw, c0, p.C, raw[e]);
        } else {
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) stage_rows(sw[i] + k, lane, piece + 512 * MB + 256 * i);
        }
      };
      ask(k0);
      for (; k0 + 32 <= p.K; k0 += D) {
        Step s;
        staged_arrived();
#pragma unroll
        for (int m = 0; m < MB; ++m) staged_row8(piece, 16 * m + l15, q, s.a[m]);
        if (NN) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int j = 0; j < NB; ++j) s.b[j][e] = raw[e][j];
        } else {
#pragma unroll
          for (int j = 0; j < NB; ++j) staged_row8(piece + 512 * MB, 16 * j + l15, q, s.b[j]);
        }
        staged_taken();
        if (k0 + D + 32 <= p.K) ask(k0 + D);
        multiply(s, clamp);
      }
    }
    for (; k0 < p.K; k0 += D) {
      Step rest;
      load(k0, p.K - k0, rest);
      multiply(rest, clamp);
    }
  };
  sweep(std::false_type());
  bool nan = false;
#pragma unroll
  for (int m = 0; m < MB; ++m) nan |= any_nan(small[m]);
  if (__ballot(nan)) sweep(std::true_type());

  __syncthreads();  // (the pieces of LDS have been read: now they take the sums)
  constexpr int EACH = BM * BN / (64 * NW) > 0 ? BM * BN / (64 * NW) : 1;
  float y[EACH];
  if (p.y) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int m = (threadIdx.x + 64 * NW * i) / BN;
      y[i] = m < BM && m0 + m < p.N && my_c < p.C ? p.y[(size_t)(m0 + m) * p.ldy + my_c] : 0.f;
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) part[wave][16 * m + 4 * q + i][NB * l15 + j] = acc[m][j][i] + small[m][j][i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int m = (threadIdx.x + 64 * NW * i) / BN;
    if (m >= BM || m0 + m >= p.N || my_c >= p.C) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += part[w][m][threadIdx.x % BN];
    float v = my_bias + sum;
    if (p.act == KH_ACT_SIGMOID) v = kh::sigmoidf(v);
    if (p.y) v = v * y[i] * (1.f - y[i]);
    p.out[(size_t)(m0 + m) * p.ldout + my_c] = v;
  }
}

// What these tiles leave to do: out += t * side of each row's adapter, then the activation or the derivative below.  A wave
// has 64 columns of a row; CHUNK rows of the stack are on their way at a time.  256 rows of rank 16: 4.9 us (four columns a
// lane, a quarter of the waves: 6.8 us; 64 rows of ranks up to 32: 4.4 and 14.0).
struct FinishArgs {
  int N, C;
  const float *t; int ldt;
  const float *side; int ldside;
  Stack st;
  const int32_t *row_adapter;
  const float *y; int ldy;
  int act;
  float *out; int ldout;
  __host__ __device__ long long units() const { return (long long)N * ((C + 63) / 64); }
};
template <int CHUNK>
__device__ __forceinline__ void finish_unit(const FinishArgs &p, long long unit, int lane) {
  const int col_units = (p.C + 63) / 64, r = (int)(unit / col_units), c = (int)(unit % col_units) * 64 + lane;
  const int cc = min(c, p.C - 1);
  float *out = p.out + (size_t)r * p.ldout + cc;
  const float *t = p.t + (size_t)r * p.ldt;
  const float raw = *out, y = p.y ? p.y[(size_t)r * p.ldy + cc] : 0.f;
  const float first = lane < CHUNK && lane < p.st.max_rank ? t[lane] : 0.f;
  const int g = __builtin_amdgcn_readfirstlane(adapter_of(p.row_adapter, p.st.num, r));
  float sum = 0.f;
  if (g >= 0) {
    int lo, rank;
    stack_rows(p.st, g, &lo, &rank);
    const float *side = p.side + (size_t)lo * p.ldside + cc;
    for (int k0 = 0; k0 < rank; k0 += CHUNK) {
      const float a = k0 == 0 ? first : lane < CHUNK && k0 + lane < rank ? t[k0 + lane] : 0.f;
      float b[CHUNK];
#pragma unroll
      for (int k = 0; k < CHUNK; ++k) b[k] = side[(size_t)min(k0 + k, rank - 1) * p.ldside];
#pragma unroll
      for (int k = 0; k < CHUNK; ++k)
        if (k0 + k < rank) sum = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), k)), b[k], sum);
    }
  }
  float v = raw + sum;
  if (p.act == KH_ACT_SIGMOID) v = kh::sigmoidf(v);
  if (p.y) v = v * y * (1.f - y);
  if (c < p.C) *out = v;
}
template <int CHUNK>
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long units = p.units();
  for (long long unit = 4ll * blockIdx.x + wave; unit < units; unit += 4ll * gridDim.x) finish_unit<CHUNK>(p, unit, lane);
}
void launch_finish(hipStream_t st, const FinishArgs &p) {
  const unsigned blocks = (unsigned)std::min((p.units() + 3) / 4, 1ll << 20);
  if (p.st.max_rank <= 16) finish_kernel<16><<<blocks, 256, 0, st>>>(p);
  else finish_kernel<32><<<blocks, 256, 0, st>>>(p);
}

// ---- the wide product, tiles through LDS ----------------------------------------------------------------------------
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v4b __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v16f mfma6_32(const Frag &a, const Frag &b, v16f c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.lo, b.hi, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.lo, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.mid, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.hi, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.mid, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.hi, c, 0, 0, 0);
  return c;
}

// four floats as three times four bfloat16
template <bool CLAMP>
__device__ __forceinline__ void split4(v4f x, v4b &hi, v4b &mid, v4b &lo) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    v2b h, m, l;
    split2_apart<CLAMP>(x[i], x[i + 1], h, m, l);
    hi[i] = h.x, hi[i + 1] = h.y;
    mid[i] = m.x, mid[i + 1] = m.y;
    lo[i] = l.x, lo[i + 1] = l.y;
  }
}

// A tile of X rows by 32 of the inner dimension lies in LDS as three images (hi, mid, lo), each of 32-row blocks of
// 4 * 32 slots of 16 bytes: slot kc * 32 + (row ^ 2 kc) holds the eight bfloat16 k = 8 kc .. 8 kc + 7 of a row, which is
// what a lane hands to the 32x32x16 instruction.  The exclusive-or puts the eight slots of two rows, which 16 lanes store at a
// time, into different banks, and leaves those of eight rows, which eight lanes load, in different ones (row ^ 4 kc: the stores
// met in pairs, 30 % of the LDS's cycles; 2 % more time for 4096 rows, 2048 -> 2048).
__device__ __forceinline__ int slot_of(int row, int kc) { return (row >> 5) * 128 + kc * 32 + ((row & 31) ^ (2 * kc)); }

// One workgroup of eight waves (WM x WN) per tile of BM x BN; a wave has MB x NB blocks of 32 x 32.  Every step of 32 of
// the inner dimension is loaded into registers two steps ahead, split there and stored to the other half of LDS while
// this step's products run; one barrier per step.  256x128 tiles, 4096 rows, 2048 -> 2048: 195 us, 176 TFLOP/s of float
// products, 1.06 PFLOP/s of bfloat16 ones (the library's fp32 product of this size: 259 us, its bfloat16 products reach 1.2
// to 1.4 PFLOP/s on this chip); products and LDS loads alone take 155 us, loading and splitting alone 95, of which 55 run
// under the former.
template <int WM, int WN, int MB, int NB, bool NN, bool VEC>
__global__ __launch_bounds__(512) void tiled_kernel(WideArgs p) {
  constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
  constexpr int A_SLOTS = BM * 4, B_SLOTS = BN * 4;
  __shared__ v8b lds[2][3][A_SLOTS + B_SLOTS];
  static_assert(WM * WN == 8 && BM % 64 == 0, "eight waves");
  constexpr int AU = BM * 8 / 512;                          // units of four floats a thread stages of X
  constexpr int BU = NN ? 0 : BN * 8 / 512;                 // of W, rows along the inner dimension
  constexpr int BC = NN ? (BN * 4 + 511) / 512 : 0;         // of W, eight floats down a column each

  // tiles in groups of four rows of tiles, the groups dealt to the dies in whole runs: a die's tiles share their operands
  const int total = p.tiles_m * p.tiles_n, per = (total + 7) / 8;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || id >= total) return;
  const int group = id / (4 * p.tiles_n), in_group = min(4, p.tiles_m - 4 * group), rest = id - group * 4 * p.tiles_n;
  const int m0 = (4 * group + rest % in_group) * BM, n0 = (rest / in_group) * BN;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, l31 = lane & 31, half = lane >> 5;

  const float *ar[AU];
#pragma unroll
  for (int u = 0; u < AU; ++u) ar[u] = p.x + (size_t)max(row_of(p.order, m0 + (tid >> 3) + 64 * u, p.N), 0) * p.ldx;
  const float *br[BU > 0 ? BU : 1];
#pragma unroll
  for (int u = 0; u < BU; ++u) br[u] = p.w + (size_t)min(n0 + (tid >> 3) + 64 * u, p.C - 1) * p.ldw;
  const int ka = (tid & 7) * 4;

  v4f ra[AU], rb[BU > 0 ? BU : 1];
  float rc[BC > 0 ? BC : 1][8];
  const float *bc[BC > 0 ? BC : 1];  // column n of W, from row 8 kc
#pragma unroll
  for (int u = 0; u < BC; ++u)
    bc[u] = p.w + (size_t)(8 * ((tid + 512 * u) / BN)) * p.ldw + min(n0 + (tid + 512 * u) % BN, p.C - 1);
  // the step at k0 into registers: a whole one, or what is left of K (zeros behind it)
  auto fetch_whole = [&](int k0) {
#pragma unroll
    for (int u = 0; u < AU; ++u) ra[u] = *reinterpret_cast<const v4f *>(ar[u] + k0 + ka);
#pragma unroll
    for (int u = 0; u < BU; ++u) rb[u] = *reinterpret_cast<const v4f *>(br[u] + k0 + ka);
#pragma unroll
    for (int u = 0; u < BC; ++u) {
      if (BC * 512 > BN * 4 && (tid + 512 * u) / BN >= 4) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) rc[u][e] = bc[u][(size_t)(k0 + e) * p.ldw];
    }
  };
  auto fetch = [&](int k0) {
    if (VEC && k0 + 32 <= p.K) return fetch_whole(k0);
#pragma unroll
    for (int u = 0; u < AU; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) ra[u][i] = k0 + ka + i < p.K ? ar[u][k0 + ka + i] : 0.f;
#pragma unroll
    for (int u = 0; u < BU; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) rb[u][i] = k0 + ka + i < p.K ? br[u][k0 + ka + i] : 0.f;
#pragma unroll
    for (int u = 0; u < BC; ++u) {
      const int kc = (tid + 512 * u) / BN;
      if (BC * 512 > BN * 4 && kc >= 4) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) rc[u][e] = k0 + 8 * kc + e < p.K ? bc[u][(size_t)(k0 + e) * p.ldw] : 0.f;
    }
  };
  auto put = [&](int buf, auto clamp) {
    const int kc = ka >> 3, sub = ka & 4;
#pragma unroll
    for (int u = 0; u < AU; ++u) {
      v4b h, m, l;
      split4<clamp.value>(ra[u], h, m, l);
      const int s = slot_of((tid >> 3) + 64 * u, kc);
      *reinterpret_cast<v4b *>(reinterpret_cast<__bf16 *>(&lds[buf][0][s]) + sub) = h;
      *reinterpret_cast<v4b *>(reinterpret_cast<__bf16 *>(&lds[buf][1][s]) + sub) = m;
      *reinterpret_cast<v4b *>(reinterpret_cast<__bf16 *>(&lds[buf][2][s]) + sub) = l;
    }
#pragma unroll
    for (int u = 0; u < BU; ++u) {
      v4b h, m, l;
      split4<clamp.value>(rb[u], h, m, l);
      const int s = A_SLOTS + slot_of((tid >> 3) + 64 * u, kc);
      *reinterpret_cast<v4b *>(reinterpret_cast<__bf16 *>(&lds[buf][0][s]) + sub) = h;
      *reinterpret_cast<v4b *>(reinterpret_cast<__bf16 *>(&lds[buf][1][s]) + sub) = m;
      *reinterpret_cast<v4b *>(reinterpret_cast<__bf16 *>(&lds[buf][2][s]) + sub) = l;
    }
#pragma unroll
    for (int u = 0; u < BC; ++u) {
      const int n = (tid + 512 * u) % BN, c = (tid + 512 * u) / BN;
      if (c < 4) {
        const Frag f = split8<clamp.value, true>(rc[u]);
        const int s = A_SLOTS + slot_of(n, c);
        lds[buf][0][s] = f.hi, lds[buf][1][s] = f.mid, lds[buf][2][s] = f.lo;
      }
    }
  };

  // hi * hi is summed apart from the five small part products: the large sum is then rounded once per instruction of its
  // own, not six times (relative error over 2048 products 3e-7 instead of 9e-7)
  v16f acc[MB][NB], rest_of[MB][NB];
  const int steps = (p.K + 31) / 32;
  // the products of one half of a step: the six part products in turn, each over all blocks (a block's sum is then
  // not waited for)
  auto multiply = [&](int buf, int h) {
    v8b fa[MB][3], fb[NB][3];
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 3; ++i) fa[m][i] = lds[buf][i][slot_of(32 * (wm * MB + m) + l31, 2 * h + half)];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 3; ++i) fb[n][i] = lds[buf][i][A_SLOTS + slot_of(32 * (wn * NB + n) + l31, 2 * h + half)];
    constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int q = 0; q < 6; ++q)
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          v16f &sum = q < 5 ? rest_of[m][n] : acc[m][n];
          sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[m][pa[q]], fb[n][pb[q]], sum, 0, 0, 0);
        }
  };
  auto sweep = [&](auto clamp) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[m][n][i] = rest_of[m][n][i] = 0.f;
    if (steps > 0) {
      fetch(0);
      put(0, clamp);
      if (steps > 1) fetch(32);
      __syncthreads();
    }
    int s = 0;
    if (VEC)
      for (; 32 * (s + 3) <= p.K; ++s) {
        const int buf = s & 1;
        multiply(buf, 0);
        put(buf ^ 1, clamp);
        fetch_whole(32 * (s + 2));
        multiply(buf, 1);
        __syncthreads();
      }
    for (; s < steps; ++s) {
      const int buf = s & 1;
      multiply(buf, 0);
      if (s + 1 < steps) put(buf ^ 1, clamp);
      if (s + 2 < steps) fetch(32 * (s + 2));
      multiply(buf, 1);
      __syncthreads();
    }
  };
  sweep(std::false_type());
  bool nan = false;
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) nan |= rest_of[m][n][i] != rest_of[m][n][i];
  if (__syncthreads_or(nan)) sweep(std::true_type());

#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[m][n] += rest_of[m][n];

  // the adapters' part, straight into registers: a wave goes through the runs of equal adapters in its rows
  const int wave_m0 = m0 + 32 * MB * wm, wave_n0 = n0 + 32 * NB * wn;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int row = lane < 32 ? row_of(p.order, wave_m0 + 32 * m + lane, p.N) : -1;
    const int my_row = __shfl(row, l31, 64);
    if (p.t) {
      const int g = adapter_of(p.row_adapter, p.st.num, row);
      const Runs runs = find_runs(g, lane);
      const float *tr = p.t + (size_t)max(my_row, 0) * p.ldt;
      for (unsigned long long left = runs.starts; left; left &= left - 1ull) {
        const int s = __builtin_ctzll(left);
        const unsigned mask = (unsigned)run_mask(runs, s);
        int lo, rank;
        stack_rows(p.st, __shfl(g, s, 64), &lo, &rank);
        v16f d[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) d[n][i] = 0.f;
        for (int k0 = 0; k0 < rank; k0 += 16) {
          float a[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = k0 + 8 * half + e < rank ? tr[k0 + 8 * half + e] : 0.f;
          const Frag fa = split8(a);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const int c = wave_n0 + 32 * n + l31;
            float b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int k = k0 + 8 * half + e;
              b[e] = k < rank && c < p.C ? p.side[(size_t)(lo + k) * p.ldside + c] : 0.f;
            }
            d[n] = mfma6_32(fa, split8(b), d[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if ((mask >> (8 * (i >> 2) + 4 * half + (i & 3))) & 1u) acc[m][n][i] += d[n][i];
      }
    }
    // out: lane l31 has a column, i counts rows
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = __shfl(row, 8 * (i >> 2) + 4 * half + (i & 3), 64);
      if (r < 0) continue;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int c = wave_n0 + 32 * n + l31;
        if (c >= p.C) continue;
        float v = acc[m][n][i];
        if (p.bias) v += p.bias[c];
        if (p.act == KH_ACT_SIGMOID) v = kh::sigmoidf(v);
        if (p.y) {
          const float yv = p.y[(size_t)r * p.ldy + c];
          v = v * yv * (1.f - yv);
        }
        p.out[(size_t)r * p.ldout + c] = v;
      }
    }
  }
}

// ---- gradients of the stacks ----------------------------------------------------------------------------------------
// g_side[begin + k, c] = sum over the rows r of an adapter of narrow[r, k] * wide[r, c].  One workgroup per adapter,
// block of 16 * NB columns and block of 16 * MB rank rows; its waves take steps of 32 rows in turn and add up in LDS.
// Both stacks in one launch.  Bound by reading `wide` once per rank block: 8192 rows of 2 x 2048, 16 adapters of up to 32: 42 us,
// 3.2 TB/s (64-column tiles, whose registers leave two waves per SIMD: 76 us); 256 rows of 40 adapters, one wave each: 6.6 us
// (eight waves, seven of them idle: 21 us).
struct GradArgs {
  const float *narrow; int ldnarrow;
  const float *wide; int ldwide; int C;
  float *grad; int ldgrad;
};
template <int MB, int NB, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW) void grad_kernel(GradArgs down, GradArgs up, int N, Stack st, const int32_t *order,
                                                       const int32_t *row_begin, int col_tiles, int rank_blocks, FinishArgs rest) {
  __shared__ float part[NW > 1 ? NW : 1][16 * MB][16 * NB];
  if (blockIdx.y >= 2u * rank_blocks) {
    const long long units = rest.units(), step = (long long)gridDim.x * (gridDim.y - 2 * rank_blocks) * NW;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (long long unit = ((long long)(blockIdx.y - 2 * rank_blocks) * gridDim.x + blockIdx.x) * NW + wave; unit < units; unit += step)
      finish_unit<16 * MB>(rest, unit, threadIdx.x & 63);
    return;
  }
  const bool is_up = blockIdx.y >= (unsigned)rank_blocks;
  const GradArgs &p = is_up ? up : down;
  const int k_base = (blockIdx.y - (is_up ? rank_blocks : 0)) * 16 * MB;
  const int g = blockIdx.x / col_tiles, n0 = (blockIdx.x % col_tiles) * 16 * NB;
  if (n0 >= p.C) return;
  int lo, rank;
  stack_rows(st, g, &lo, &rank);
  if (k_base >= rank) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, q = lane >> 4;
  const int begin = min(max(row_begin[g], 0), N), end = min(row_begin[g + 1], N), c0 = n0 + NB * l15;
  v4f acc[MB][NB], small[MB][NB];
  auto sweep = [&](auto clamp) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[m][j] = small[m][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    int mine = begin + 32 * wave + lane < end && lane < 32 ? row_of(order, begin + 32 * wave + lane, N) : -1;
    for (int r0 = begin + 32 * wave; r0 < end; r0 += 32 * NW) {
      float a[MB][8], b[NB][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = __shfl(mine, inner(q, e), 64);
#pragma unroll
        for (int m = 0; m < MB; ++m)
          a[m][e] = r >= 0 && k_base + 16 * m + l15 < rank ? p.narrow[(size_t)r * p.ldnarrow + k_base + 16 * m + l15] : 0.f;
        float v[NB] = {};
        if (r >= 0) load_cols<NB, VEC>(p.wide + (size_t)r * p.ldwide, c0, p.C, v);
#pragma unroll
        for (int j = 0; j < NB; ++j) b[j][e] = v[j];
      }
      const int later = r0 + 32 * NW + lane;
      mine = later < end && lane < 32 ? row_of(order, later, N) : -1;
      Frag fa[MB];
#pragma unroll
      for (int m = 0; m < MB; ++m) fa[m] = split8<clamp.value>(a[m]);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const Frag fb = split8<clamp.value>(b[j]);
#pragma unroll
        for (int m = 0; m < MB; ++m) mfma6(fa[m], fb, acc[m][j], small[m][j]);
      }
    }
  };
  sweep(std::false_type());
  bool nan = false;
#pragma unroll
  for (int m = 0; m < MB; ++m) nan |= any_nan(small[m]);
  if (__ballot(nan)) sweep(std::true_type());
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[m][j] += small[m][j];
  if (NW == 1) {  // nothing to add up
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int k = k_base + 16 * m + 4 * q + i;
          if (k < rank && c0 + j < p.C) p.grad[(size_t)(lo + k) * p.ldgrad + c0 + j] = acc[m][j][i];
        }
    return;
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) part[wave][16 * m + 4 * q + i][NB * l15 + j] = acc[m][j][i];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * MB * NB; e += 64 * NW) {
    const int k = e / (16 * NB), c = e % (16 * NB);
    if (k_base + k >= rank || n0 + c >= p.C) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += part[w][k][c];
    p.grad[(size_t)(lo + k_base + k) * p.ldgrad + n0 + c] = v;
  }
}
template <int MB, int NW, bool VEC>
void launch_grad(hipStream_t st, const GradArgs &down, const GradArgs &up, int N, const Stack &stack, const int32_t *order,
                 const int32_t *row_begin, int col_tiles, const FinishArgs &rest) {
  const int rank_blocks = (stack.max_rank + 16 * MB - 1) / (16 * MB);
  const long long x = (long long)col_tiles * stack.num, more = (rest.units() + x * NW - 1) / (x * NW);
  const dim3 grid((unsigned)x, 2 * rank_blocks + (unsigned)std::min(more, 60000ll));
  grad_kernel<MB, 2, NW, VEC><<<grid, 64 * NW, 0, st>>>(down, up, N, stack, order, row_begin, col_tiles, rank_blocks, rest);
}
template <bool VEC>
void launch_grads(hipStream_t st, const GradArgs &down, const GradArgs &up, int N, const Stack &stack, const int32_t *order,
                  const int32_t *row_begin, int col_tiles, const FinishArgs &rest) {
  // one wave for adapters of few rows
  const bool few = N <= 64 * (long long)stack.num;
  if (stack.max_rank <= 16) {
    if (few) launch_grad<1, 1, VEC>(st, down, up, N, stack, order, row_begin, col_tiles, rest);
    else launch_grad<1, 8, VEC>(st, down, up, N, stack, order, row_begin, col_tiles, rest);
  } else {
    if (few) launch_grad<2, 1, VEC>(st, down, up, N, stack, order, row_begin, col_tiles, rest);
    else launch_grad<2, 8, VEC>(st, down, up, N, stack, order, row_begin, col_tiles, rest);
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------
bool vec_ok(const float *p, int ld) { return p == nullptr || (kh::aligned16(p) && ld % 4 == 0); }

Stack stack_of(const khAdapters &ad) {
  Stack st = {ad.num, ad.max_rank, ad.rows, ad.begin, ad.scale};
  return st;
}

int narrow_window(int N) {
  // windows of 16 rows fill the matrix instruction; below 256 of them (one per compute unit) smaller ones are faster
  int window = 16;
  while (window > 1 && (N + window - 1) / window < 256) window /= 2;
  return window;
}
template <bool VEC>
void launch_narrow(hipStream_t st, const NarrowArgs &p) {
  const int nb = p.st.max_rank <= 16 ? 1 : 2;
  const dim3 grid((p.N + p.window - 1) / p.window, (p.st.max_rank + 16 * nb - 1) / (16 * nb));
  if (nb == 1) narrow_kernel<1, VEC><<<grid, 64 * kNarrowWaves, 0, st>>>(p);
  else narrow_kernel<2, VEC><<<grid, 64 * kNarrowWaves, 0, st>>>(p);
}

// The blocks of the narrow product in front of small tiles.  (a multiple of 8, so that the tiles still meet their dies; the blocks
// too many are behind the last rank column)
unsigned narrow_blocks_of(const WideArgs &p, const NarrowArgs &narrow) {
  if (p.t == nullptr) return 0;
  const int fn = p.st.max_rank <= 16 ? 1 : 2, windows = (p.N + narrow.window - 1) / narrow.window;
  return (unsigned)(windows * ((p.st.max_rank + 16 * fn - 1) / (16 * fn)) + 7) / 8 * 8;
}
template <int MB, int NB, int NW, bool NN, bool VEC>
void launch_wide_tile(hipStream_t st, WideArgs p, const NarrowArgs &narrow, FinishArgs *rest) {
  p.tiles_m = (p.N + 16 * MB - 1) / (16 * MB);
  p.tiles_n = (p.C + 16 * NB - 1) / (16 * NB);
  const unsigned blocks = 8u * ((p.tiles_n + 7) / 8) * (unsigned)p.tiles_m;
  if (p.t == nullptr) return wide_kernel<MB, NB, NW, NN, VEC, 0><<<blocks, 64 * NW, 0, st>>>(p, narrow, 0, 0);
  *rest = {p.N, p.C, p.t, p.ldt, p.side, p.ldside, p.st, p.row_adapter, p.y, p.ldy, p.act, p.out, p.ldout};
  p.y = nullptr, p.act = KH_ACT_NONE;
  const int windows = (p.N + narrow.window - 1) / narrow.window, narrow_blocks = (int)narrow_blocks_of(p, narrow);
  if (p.st.max_rank <= 16) wide_kernel<MB, NB, NW, NN, VEC, 1><<<narrow_blocks + blocks, 64 * NW, 0, st>>>(p, narrow, windows, narrow_blocks);
  else wide_kernel<MB, NB, NW, NN, VEC, 2><<<narrow_blocks + blocks, 64 * NW, 0, st>>>(p, narrow, windows, narrow_blocks);
}
template <int WM, int WN, int MB, int NB, bool NN, bool VEC>
void launch_tiled(hipStream_t st, WideArgs p) {
  p.tiles_m = (p.N + 32 * MB * WM - 1) / (32 * MB * WM);
  p.tiles_n = (p.C + 32 * NB * WN - 1) / (32 * NB * WN);
  const unsigned blocks = 8u * (((unsigned)p.tiles_m * p.tiles_n + 7) / 8);
  tiled_kernel<WM, WN, MB, NB, NN, VEC><<<blocks, 512, 0, st>>>(p);
}
// Which kernel and tile.  The tiles of a product are worked off in rounds of one per compute unit; what a round takes of a
// whole call was fitted to calls of 1 to 4096 rows with adapters of rank 16, 512 to 2048 inner indices and columns (us): 16 rows
// x 16 columns 7, 16 x 32 11, 32 x 64 21, 64 x 128 62, 128 x 128 95, 256 x 128 170; the choice is within 1.3 % of the fastest
// tile on average, within 14 % at worst.  E.g. 2048 -> 2048: 1 row 16x16 10 us (16x32 10, 32x64 18); 64 rows 16x32 16 (16x16 16,
// 32x64 20); 256 rows 32x64 28 (16x32 38, 64x128 66); 1024 rows 64x128 73 (32x64 85, 128x128 101); 2048 rows 128x128 114 (64x128
// 121, 256x128 167); 4096 rows 256x128 193 (128x128 220).
template <bool NN, bool VEC>
int launch_wide(hipStream_t st, const WideArgs &p, const NarrowArgs &narrow, FinishArgs *rest) {
  static const struct { int rows, cols, round, threads; } kTiles[] = {{16, 16, 7, 512}, {16, 32, 11, 1024}, {32, 64, 21, 512},
                                                                      {64, 128, 62, 512}, {128, 128, 95, 512}, {256, 128, 170, 512}};
  // (hipK_gemm_row_invariant: the tiled kernels only, which sum an element in the same order whatever their tile; so too where
  // the narrow product's workgroups might be too many in front of small tiles)
  const int first = kh::gemm_row_invariant() || p.N > (1 << 20) ? 3 : 0;
  int best = -1;
  long long least = 0;
  for (int i = first; i < 6; ++i) {
    const long long tiles_n = (p.C + kTiles[i].cols - 1) / kTiles[i].cols, tiles_m = (p.N + kTiles[i].rows - 1) / kTiles[i].rows;
    const long long tiles = tiles_m * tiles_n, cost = (tiles + 255) / 256 * kTiles[i].round;
    // a grid counts its threads in 32 bits (more are cut off without an error)
    const long long blocks = i > 2 ? (tiles + 7) / 8 * 8 : (tiles_n + 7) / 8 * 8 * tiles_m + narrow_blocks_of(p, narrow);
    if (blocks * kTiles[i].threads > 0xffffffffll) continue;
    if (best < 0 || cost < least) best = i, least = cost;
  }
  if (best < 0) {
    snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "%d rows of %d columns: too many tiles", p.N, p.C);
    return KH_ERR_TOO_LARGE;
  }
  if (best > 2 && p.t) launch_narrow<VEC>(st, narrow);
  switch (best) {
    case 0: launch_wide_tile<1, 1, 8, NN, VEC>(st, p, narrow, rest); break;
    case 1: launch_wide_tile<1, 2, 16, NN, VEC>(st, p, narrow, rest); break;
    case 2: launch_wide_tile<2, 4, 8, NN, VEC>(st, p, narrow, rest); break;
    case 3: launch_tiled<2, 4, 1, 1, NN, VEC>(st, p); break;
    case 4: launch_tiled<4, 2, 1, 2, NN, VEC>(st, p); break;
    default: launch_tiled<4, 2, 2, 2, NN, VEC>(st, p);
  }
  return kh::launch_status();
}

// A grid counts its threads in 32 bits: 2^26 rows in windows of 16 rows and 512 threads fill half of that.
constexpr int kMaxRows = 1 << 26, kMaxAdapters = 1 << 21, kMaxDim = 1 << 30;
int too_many(const char *what, int n, int most) {
  snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "%d %s: at most %d", n, what, most);
  return KH_ERR_TOO_LARGE;
}

int check_adapters(const khAdapters *ad, const int32_t *row_adapter, int32_t N, int32_t I, int32_t O) {
  KH_REQUIRE(ad != nullptr && ad->num >= 0);
  if (N > kMaxRows) return too_many("rows", N, kMaxRows);
  if (std::max(I, O) > kMaxDim) return too_many("columns", std::max(I, O), kMaxDim);  // (counted in 32 bits, a step further)
  if (ad->num == 0) return KH_OK;
  KH_REQUIRE(ad->max_rank >= 1 && ad->rows >= 0);
  if (ad->max_rank > KH_MAX_ADAPTER_RANK) {
    snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "adapters of rank %d: at most %d", ad->max_rank,
             KH_MAX_ADAPTER_RANK);
    return KH_ERR_TOO_LARGE;
  }
  KH_REQUIRE(ad->begin != nullptr && (N == 0 || row_adapter != nullptr));
  KH_REQUIRE(ad->rows == 0 || (ad->down != nullptr && ad->up != nullptr));
  KH_REQUIRE(ad->lddown >= I && ad->ldup >= O);
  return KH_OK;
}

// the library works on the device that hipK_init chose
int check_device() {
  int now = -1;
  KH_HIP(hipGetDevice(&now));
  KH_REQUIRE(now == kh::ctx().device);
  return KH_OK;
}

}  // namespace

KH_EXPORT int hipI32_adapter_plan(khStream_t s, const int32_t *row_adapter, int32_t N, int32_t num, int32_t *order,
                                  int32_t *row_begin) {
  KH_REQUIRE(N >= 0 && num >= 0 && row_begin != nullptr);
  KH_REQUIRE(N == 0 || (row_adapter != nullptr && order != nullptr));
  if (N > kMaxRows) return too_many("rows", N, kMaxRows);  // (counted in 32 bits, a workgroup's 1024 further)
  if (num > kMaxAdapters) return too_many("adapters", num, kMaxAdapters);  // (a workgroup of up to 1024 for each)
  // every workgroup reads all ids, twice: 2^40 of them are 8 TB out of the caches, about a second
  if (N * (num + 1ll) > 1ll << 40) {
    snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "%d rows of %d adapters: too many together", N, num);
    return KH_ERR_TOO_LARGE;
  }
  int rc = kh::check_apart(__func__, {{"order", order, 1, N, N}, {"row_begin", row_begin, 1, num + 1ll, num + 1ll}},
                           {{"row_adapter", row_adapter, 1, N, N}});
  if (rc != KH_OK) return rc;
  KH_CHECK_INIT();
  rc = check_device();
  if (rc != KH_OK) return rc;
  const int threads = N <= 256 ? 256 : 1024;
  plan_kernel<<<(unsigned)num + 1u, threads, 0, kh::pick(s)>>>(row_adapter, N, num, order, row_begin);
  return kh::launch_status();
}

KH_EXPORT int hipF_adapter_forward(khStream_t s, int act, int32_t N, int32_t O, int32_t I, const float *in, int32_t ldin,
                                   const float *W, int32_t ldw, const float *bias, const khAdapters *ad,
                                   const int32_t *row_adapter, const int32_t *order, float *t, int32_t ldt, float *out,
                                   int32_t ldout) {
  KH_REQUIRE(act == KH_ACT_NONE || act == KH_ACT_SIGMOID || act == KH_ACT_SOFTMAX);
  KH_REQUIRE(N >= 0 && O >= 0 && I >= 0);
  int rc = check_adapters(ad, row_adapter, N, I, O);
  if (rc != KH_OK) return rc;
  KH_REQUIRE(N == 0 || (ldin >= I && ldw >= I && ldout >= O));
  KH_REQUIRE(ad->num == 0 || N == 0 || (t != nullptr && ldt >= ad->max_rank));
  KH_REQUIRE(N == 0 || O == 0 || (out != nullptr && (I == 0 || (in != nullptr && W != nullptr))));
  const int num = ad->num, stack_rows = num > 0 ? ad->rows : 0;
  rc = kh::check_apart(__func__, {{"out", out, N, O, ldout}, {"t", num > 0 ? t : nullptr, N, ad->max_rank, ldt}},
                       {{"in", in, N, I, ldin}, {"W", W, O, I, ldw}, {"bias", bias, 1, O, O},
                        {"down", ad->down, stack_rows, I, ad->lddown}, {"up", ad->up, stack_rows, O, ad->ldup},
                        {"begin", ad->begin, num > 0, num + 1ll, num + 1ll}, {"scale", ad->scale, num > 0, num, num},
                        {"row_adapter", row_adapter, num > 0, N, N}, {"order", order, 1, N, N}});
  if (rc != KH_OK) return rc;
  KH_CHECK_INIT();
  rc = check_device();
  if (rc != KH_OK) return rc;
  if (N == 0 || O == 0) return KH_OK;
  hipStream_t st = kh::pick(s);
  const Stack stack = stack_of(*ad);
  const bool vec = vec_ok(in, ldin) && vec_ok(W, ldw) && (ad->num == 0 || (vec_ok(ad->down, ad->lddown) &&
                   vec_ok(ad->up, ad->ldup) && vec_ok(t, ldt)));
  const NarrowArgs na = {in, ldin, N, I, ad->down, ad->lddown, stack, row_adapter, order, narrow_window(N), t, ldt};
  WideArgs p = {in, ldin, W, ldw, N, I, O, bias, ad->num > 0 ? t : nullptr, ldt, ad->up, ad->ldup, stack, row_adapter, order,
                nullptr, 0, act, out, ldout, 0, 0};
  FinishArgs rest = {};
  rc = vec ? launch_wide<false, true>(st, p, na, &rest) : launch_wide<false, false>(st, p, na, &rest);
  if (rc != KH_OK) return rc;
  if (rest.N > 0) launch_finish(st, rest);
  rc = kh::launch_status();
  if (rc != KH_OK || act != KH_ACT_SOFTMAX) return rc;
  const MatrixDim d = {N, O, ldout};
  return hipF_softmax(s, out, out, d);
}

KH_EXPORT int hipF_adapter_backward(khStream_t s, int32_t N, int32_t O, int32_t I, const float *e, int32_t lde,
                                    const float *in, int32_t ldin, const float *W, int32_t ldw, const khAdapters *ad,
                                    const int32_t *row_adapter, const int32_t *order, const int32_t *row_begin,
                                    const float *t, int32_t ldt, float *u, int32_t ldu, const float *y, int32_t ldy,
                                    float *eout, int32_t ldeout, float *gdown, int32_t ldgdown, float *gup,
                                    int32_t ldgup) {
  KH_REQUIRE(N >= 0 && O >= 0 && I >= 0);
  int rc = check_adapters(ad, row_adapter, N, I, O);
  if (rc != KH_OK) return rc;
  const bool grads = ad->num > 0 && (gdown != nullptr || gup != nullptr);
  const int cols = grads && ad->rows > 0 ? std::max(gdown != nullptr ? I : 0, gup != nullptr ? O : 0) : 0;
  const int col_tiles = (cols + 31) / 32;
  KH_REQUIRE(N == 0 || O == 0 || (e != nullptr && lde >= O));
  KH_REQUIRE(eout == nullptr || (W != nullptr && ldw >= I && ldeout >= I && (y == nullptr || ldy >= I)));
  KH_REQUIRE(ad->num == 0 || N == 0 || (u != nullptr && ldu >= ad->max_rank));
  KH_REQUIRE(!grads || (row_begin != nullptr && (N == 0 || order != nullptr)));
  KH_REQUIRE(gdown == nullptr || (ldgdown >= I && (N == 0 || (in != nullptr && ldin >= I))));
  KH_REQUIRE(gup == nullptr || (ldgup >= O && (N == 0 || (t != nullptr && ldt >= ad->max_rank))));
  if ((long long)col_tiles * ad->num > 0x7fffffLL) {  // (workgroups of up to 512: the grid counts threads in 32 bits)
    snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "gradients of %d adapters of %d columns: too many", ad->num, cols);
    return KH_ERR_TOO_LARGE;
  }
  // (what a call does not read or write may be anywhere)
  const int num = ad->num, stack_rows = num > 0 ? ad->rows : 0, grad_rows = grads ? stack_rows : 0;
  rc = kh::check_apart(__func__,
                       {{"u", num > 0 ? u : nullptr, N, ad->max_rank, ldu}, {"eout", eout, N, I, ldeout},
                        {"gdown", gdown, grad_rows, I, ldgdown}, {"gup", gup, grad_rows, O, ldgup}},
                       {{"e", e, N, O, lde}, {"in", gdown ? in : nullptr, N, I, ldin}, {"W", eout ? W : nullptr, O, I, ldw},
                        {"y", eout ? y : nullptr, N, I, ldy}, {"t", gup ? t : nullptr, N, ad->max_rank, ldt},
                        {"down", ad->down, eout ? stack_rows : 0, I, ad->lddown}, {"up", ad->up, stack_rows, O, ad->ldup},
                        {"begin", ad->begin, num > 0, num + 1ll, num + 1ll}, {"scale", ad->scale, num > 0, num, num},
                        {"row_adapter", row_adapter, num > 0, N, N}, {"order", order, 1, N, N},
                        {"row_begin", row_begin, grads, num + 1ll, num + 1ll}});
  if (rc != KH_OK) return rc;
  KH_CHECK_INIT();
  rc = check_device();
  if (rc != KH_OK) return rc;
  hipStream_t st = kh::pick(s);
  const Stack stack = stack_of(*ad);
  const NarrowArgs na = {e, lde, N, O, ad->up, ad->ldup, stack, row_adapter, order, narrow_window(N), u, ldu};
  if (ad->num > 0 && N > 0 && (eout == nullptr || I == 0)) {
    if (vec_ok(e, lde) && vec_ok(ad->up, ad->ldup)) launch_narrow<true>(st, na);
    else launch_narrow<false>(st, na);
    rc = kh::launch_status();
    if (rc != KH_OK) return rc;
  }
  FinishArgs rest = {};
  if (eout != nullptr && N > 0 && I > 0) {
    WideArgs p = {e, lde, W, ldw, N, O, I, nullptr, ad->num > 0 ? u : nullptr, ldu, ad->down, ad->lddown, stack, row_adapter,
                  order, y, ldy, KH_ACT_NONE, eout, ldeout, 0, 0};
    const bool vec = vec_ok(e, lde) && vec_ok(W, ldw) && (ad->num == 0 || (vec_ok(ad->down, ad->lddown) &&
                     vec_ok(ad->up, ad->ldup) && vec_ok(u, ldu)));
    rc = vec ? launch_wide<true, true>(st, p, na, &rest) : launch_wide<true, false>(st, p, na, &rest);
    if (rc != KH_OK) return rc;
  }
  if (cols == 0) {
    if (rest.N > 0) launch_finish(st, rest);
    return kh::launch_status();
  }
  GradArgs gd = {u, ldu, in, ldin, gdown != nullptr ? I : 0, gdown, ldgdown};
  GradArgs gu = {t, ldt, e, lde, gup != nullptr ? O : 0, gup, ldgup};
  const bool vec = (gdown == nullptr || vec_ok(in, ldin)) && (gup == nullptr || vec_ok(e, lde));
  if (vec) launch_grads<true>(st, gd, gu, N, stack, order, row_begin, col_tiles, rest);
  else launch_grads<false>(st, gd, gu, N, stack, order, row_begin, col_tiles, rest);
  return kh::launch_status();
}
