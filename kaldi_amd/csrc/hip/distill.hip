// Learning from another network's outputs: hipF_row_top (a row's largest logits) and hipF_distill_eval (loss and gradient
// towards them, mixed with hard labels); include/kaldi_hip.h has the formulas.
//
// A row is one workgroup's, whose threads hold up to kHold floats of it each: up to 1024 * kHold = 20480 columns stay in
// registers between the maximum, the sum and the output, so that the logits are read (and their gradient written) once.  Longer
// rows are gone through in such chunks, by hipF_row_top once, by hipF_distill_eval with a gradient twice: the sums have to be
// whole before the first column can be written.
//
// Memory rates that the figures below compare with (calls in a row, operands in turn that the last-level cache does not hold):
// this library's column sums read 0.3 to 4 GB at 5.9 to 6.0 TB/s, its sigmoid copies 300 to 600 MB at 6.2 and 2 to 4 GB at 5.1.
#include <algorithm>

#include "common.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
constexpr int kHold = 20;  // floats of the row per thread: five 16-byte loads

// exp(c * x) for c = log2(e) * const given as the sum of two floats: the product's rounding error is carried along, so
// the result is good to two units in the last place wherever it is a normal number.
struct ExpScale {
  float hi, lo;
};
__device__ __forceinline__ float exp_scaled(float x, ExpScale c) {
  const float a = x * c.hi;
  const float b = __builtin_fmaf(x, c.lo, __builtin_fmaf(x, c.hi, -a));
  const float e = __builtin_amdgcn_exp2f(a);
  // (an exp2 of 0 or inf stays what it is: b is not finite there)
  return a < -150.f ? 0.f : __builtin_fmaf(e, b * 0.693147180559945309f, e);
}
ExpScale exp_scale(double times) {
  const double c = 1.44269504088896340736 * times;
  ExpScale s;
  s.hi = (float)c;
  s.lo = (float)(c - (double)s.hi);
  return s;
}

// Columns of the chunk that begins at c0, as thread `tid` of THREADS holds them: element i of the array is column
// column_of(i).  Neighbouring threads load neighbouring 16 bytes where the row allows it.
template <int THREADS, bool VEC>
__device__ __forceinline__ int column_of(int c0, int tid, int i) {
  return VEC ? c0 + ((i >> 2) * THREADS + tid) * 4 + (i & 3) : c0 + i * THREADS + tid;
}
// a chunk of the row in registers, -inf behind the row's end
template <int THREADS, bool VEC>
__device__ __forceinline__ void read_chunk(const float *row, int c0, int C, int tid, float (&z)[kHold]) {
  constexpr int w = VEC ? 4 : 1;
#pragma unroll
  for (int i = 0; i < kHold; i += w) {
    const int c = column_of<THREADS, VEC>(c0, tid, i);
    if (VEC && c + 4 <= C) {
      const v4f v = *reinterpret_cast<const v4f *>(row + c);
      z[i] = v.x, z[(i + 1) % kHold] = v.y, z[(i + 2) % kHold] = v.z, z[(i + 3) % kHold] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < w; ++j) z[i + j] = c + j < C ? row[c + j] : -INFINITY;
    }
  }
}
// what lies behind the row's end becomes -inf
template <int THREADS, bool VEC>
__device__ __forceinline__ void end_chunk(unsigned left, int tid, float (&z)[kHold]) {
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int w = VEC ? 4 : 1;
#pragma unroll
  for (int i = 0; i < kHold; i += w)
    if (left < (unsigned)((i / w) * THREADS + 64 * wave + 64) * w)  // (a wave whose columns are all there has nothing to do)
#pragma unroll
      for (int j = 0; j < w; ++j)
        if (column_of<THREADS, VEC>(0, tid, i + j) >= (int)left) z[i + j] = -INFINITY;
}

// Reductions over a wave in six steps of cross-lane operands (within rows of 16 lanes, then from row to row); every lane
// gets the result, as a scalar.
template <int CTRL, int ROWS>
__device__ __forceinline__ float lanes(float otherwise, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(otherwise), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_add(float v) {
  v += lanes<0x111, 0xf>(0.f, v);  // row_shr:1, 2, 4, 8
  v += lanes<0x112, 0xf>(0.f, v);
  v += lanes<0x114, 0xf>(0.f, v);
  v += lanes<0x118, 0xf>(0.f, v);
  v += lanes<0x142, 0xa>(0.f, v);  // row_bcast:15, 31
  v += lanes<0x143, 0xc>(0.f, v);
  return last_lane(v);
}
__device__ __forceinline__ float wave_most(float v) {  // (passes over NaN, as fmaxf does)
  v = fmaxf(v, lanes<0x111, 0xf>(-INFINITY, v));
  v = fmaxf(v, lanes<0x112, 0xf>(-INFINITY, v));
  v = fmaxf(v, lanes<0x114, 0xf>(-INFINITY, v));
  v = fmaxf(v, lanes<0x118, 0xf>(-INFINITY, v));
  v = fmaxf(v, lanes<0x142, 0xa>(-INFINITY, v));
  v = fmaxf(v, lanes<0x143, 0xc>(-INFINITY, v));
  return last_lane(v);
}

// 16 (VEC) or 4 bytes per lane straight into LDS: lane l's land at `to` + l * size, `to` the same for the whole wave
template <bool VEC>
__device__ __forceinline__ void load_to_lds(const float *from, float *to) {
  typedef __attribute__((address_space(1))) const void gvoid;
  typedef __attribute__((address_space(3))) void lvoid;
  if constexpr (VEC) __builtin_amdgcn_global_load_lds((gvoid *)from, (lvoid *)to, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds((gvoid *)from, (lvoid *)to, 4, 0, 0);
}
// A chunk of `left` columns (or the first THREADS * kHold of them) into LDS, every wave its own part; what a lane gets for
// a column behind the row's end is some column of it.  Loads are not guarded one by one but moved back to the row's last 16
// bytes, which begin inside the row: an aligned load that begins inside an allocation stays in its page.
template <int THREADS, bool VEC>
__device__ __forceinline__ void load_chunk(const float *from, int left, float *lds, int tid, int wave) {
  constexpr int w = VEC ? 4 : 1;
  const unsigned last = VEC ? (unsigned)(left - 1) & ~3u : (unsigned)(left - 1);
#pragma unroll
  for (int i = 0; i < kHold / w; ++i)
    load_to_lds<VEC>(from + min((unsigned)(i * THREADS + tid) * w, last), lds + (i * THREADS + wave * 64) * w);
}
// ... and from there into registers; afterwards the place may be loaded into again
template <int THREADS, bool VEC>
__device__ __forceinline__ void take_chunk(const float *lds, int tid, float (&z)[kHold]) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part has arrived
#pragma unroll
  for (int i = 0; i < kHold; ++i) z[i] = lds[column_of<THREADS, VEC>(0, tid, i)];
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and has been read
}

// ---- the K largest of a row -------------------------------------------------------------------------------------------
// Order of the answer: by value, NaN above everything, -0 = +0, then by ascending column.  ordered() makes the float's
// bits monotone; a 64-bit key with the complement of the column below them has the whole order.
typedef unsigned long long key_t;
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned b = __float_as_uint(x + 0.f);  // -0 + 0 = +0
  const unsigned u = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : u;
}
__device__ __forceinline__ float unordered(unsigned u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ key_t key_of(float x, int c) { return (key_t)ordered(x) << 32 | (unsigned)~c; }

constexpr int kCap = 1024;  // candidates of a chunk, next to the KH_MAX_TOP of the chunks before

// AHEAD false: a workgroup has one row, of one chunk; 64 registers, so that eight waves share a SIMD and hide each other's
// loads (4096 rows of 9000, K 32: 36.7 us, 4.0 TB/s, two thirds of what column sums read at; the vector units are busy for 56 % of
// that, and a workgroup asks for nothing more while it works on its row).  AHEAD: rows of several
// chunks of equal length; a workgroup takes one row after another and has the next chunk loaded into LDS while it works on one
// in registers, a wave waiting for its own part only (256 rows of 70001, K 64: 24.1 us, 25.0 with whole chunks and a rest;
// short rows measure 44 us that way).
// A row's first chunk: its threads form G groups; a value that at least K groups' maxima reach is a lower bound of the
// chunk's K-th largest, and where large values are spread over the row few more than K elements reach the best such value.
// It is found by bisection to K .. 1.25 K groups, every wave for itself.  (Later chunks: the K-th largest so far.)  The
// elements that reach the bound are collected in LDS and ranked by counting; the K largest are kept.  Where more than kCap reach the bound (large values crowded into few groups, many equal ones), and
// where the chunk holds a NaN or +inf, or fewer than K groups a number, a bound on the distinct keys is found by bisection over
// the chunk, which is read again from the caches in every round.  That is slow: 4096 rows of 9000, K 32, of one value or nearly all
// -inf 1.4 ms, of eight values 0.56 ms, with one NaN or +inf each 0.12 ms, in ascending order (no search) 66 us; 256 rows of 70001, K 64:
// 0.77 to 0.80 ms, 0.73 ms, 47 us, 0.19 ms.
template <int THREADS, bool VEC, bool AHEAD>
__global__ __launch_bounds__(THREADS, AHEAD ? 4 : THREADS == 64 ? 3 : 8) void row_top_kernel(const float *mat, MatrixDim d, int K, int32_t *idx, int ldidx,
                                                          float *val, int ldval, float *lse) {
  constexpr int G = THREADS < 256 ? THREADS : 256, per = THREADS / G, waves = THREADS / 64, chunk = THREADS * kHold;
  __shared__ __align__(16) float ahead[AHEAD ? chunk : 4];
  __shared__ __align__(16) key_t cand[kCap + KH_MAX_TOP];
  __shared__ key_t best[KH_MAX_TOP];
  __shared__ float gmax[G];
  __shared__ float max_s[waves], sum_s[waves];
  __shared__ int count_s[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // chunks of equal length
  const int chunks = (d.cols + chunk - 1) / chunk, step = AHEAD && chunks > 1 ? ((d.cols + chunks - 1) / chunks + 3) & ~3 : chunk;
  if (AHEAD && blockIdx.x < (unsigned)d.rows && d.cols > 0)
    load_chunk<THREADS, VEC>(mat + (size_t)blockIdx.x * d.stride, min(d.cols, step), ahead, tid, wave);
  for (long long r = blockIdx.x; r < d.rows; r += gridDim.x) {
    const float *row = mat + (size_t)r * d.stride;
    int have = 0;          // valid entries of best[]
    float m = -INFINITY;   // this wave's maximum and sum of exp(x - m)
    float sum = 0.f;
    if (tid == 0) count_s[0] = 0;
    int turn = 0;
    for (int c0 = 0; c0 < d.cols; c0 += step, turn ^= 1) {
      float z[kHold];
      int t = tid;  // (columns are worked out where they are needed: hidden from the compiler, which would keep 20 of them)
      asm volatile("" : "+v"(t));
      if (AHEAD) {
        take_chunk<THREADS, VEC>(ahead, tid, z);
        const int left = d.cols - c0;
        if (left > step) load_chunk<THREADS, VEC>(row + c0 + step, min(left - step, step), ahead, tid, wave);
        else if (r + gridDim.x < d.rows) load_chunk<THREADS, VEC>(row + (size_t)gridDim.x * d.stride, min(d.cols, step), ahead, tid, wave);
        end_chunk<THREADS, VEC>(min(left, step), t, z);
      } else {
        read_chunk<THREADS, VEC>(row, c0, d.cols, t, z);
      }
      float mine = z[0];
#pragma unroll
      for (int i = 1; i < kHold; ++i) mine = fmaxf(mine, z[i]);
      const bool first = have < K;
      if (first) {
        float of_group = mine;
#pragma unroll
        for (int o = per / 2; o > 0; o >>= 1) of_group = fmaxf(of_group, __shfl_xor(of_group, o, 64));
        if (tid % per == 0) gmax[tid / per] = of_group;
        __syncthreads();
      }
      // the wave's sum; also what tells of a NaN or +inf
      const float top = fmaxf(m, wave_most(mine));
      const float base = top == -INFINITY ? 0.f : top;
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < kHold; ++i) part += __builtin_amdgcn_exp2f((z[i] - base) * 1.44269504088896340736f);
      part = wave_add(part);
      sum = (sum == 0.f ? 0.f : sum * __builtin_amdgcn_exp2f((m - base) * 1.44269504088896340736f)) + part;
      m = top;
      float bound = first ? -INFINITY : unordered((unsigned)(best[K - 1] >> 32));
      if (tid < have) cand[tid] = best[tid];
      int n = 0;
      // Collect with the K-th largest of the chunks before as the bound; where there is none, and where that lets too many
      // through, with the groups'.
      for (int attempt = first ? 1 : 0; attempt < 2; ++attempt) {
        bool none = part != part;  // nothing to collect here (this wave's NaN sends all to the search below)
        if (attempt) {
          if (!first) {
            float of_group = mine;
#pragma unroll
            for (int o = per / 2; o > 0; o >>= 1) of_group = fmaxf(of_group, __shfl_xor(of_group, o, 64));
            if (tid % per == 0) gmax[tid / per] = of_group;
            __syncthreads();
          }
          float g[G / 64];
#pragma unroll
          for (int j = 0; j < G / 64; ++j) g[j] = gmax[lane + 64 * j];
          float most = g[0], least = g[0];
#pragma unroll
          for (int j = 1; j < G / 64; ++j) most = fmaxf(most, g[j]), least = fminf(least, g[j]);
          // `low` is reached by at least K groups (K <= G), `high` by fewer, or it is the largest of all.  What is behind
          // the row's end counts as -inf: no bound is the worse for it.
          unsigned low = ordered(-wave_most(-least)), high = ordered(wave_most(most));
          for (int round = 0; round < 32 && high - low > 1u; ++round) {
            const unsigned mid = low + (high - low) / 2;
            const float at = unordered(mid);
            int reach = 0;
#pragma unroll
            for (int j = 0; j < G / 64; ++j) reach += __popcll(__ballot(g[j] >= at));
            if (reach >= K) {
              low = mid;
              if (reach <= K + (K >> 2)) break;
            } else {
              high = mid;
            }
          }
          bound = fmaxf(bound, unordered(low));
          none |= !(bound > -INFINITY);  // (it would let in what is behind the row's end)
        }
        // one place in the list per wave, then places by counting
        int hits = 0;
#pragma unroll
        for (int i = 0; i < kHold; ++i) hits += __popcll(__ballot(z[i] >= bound));
        if (none) hits = 1 << 20;
        if (hits) {
          int at = 0;
          if (lane == 0) at = atomicAdd(&count_s[turn], hits);
          at = __builtin_amdgcn_readfirstlane(at) + have;
          float limit = bound;
          asm volatile("" : "+v"(limit), "+v"(t));  // (compared anew: 20 masks would not fit the scalar registers)
          if (!none) {
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
              const unsigned long long hit = __ballot(z[i] >= limit);
              if (hit) {
                const int place = at + __builtin_amdgcn_mbcnt_hi((unsigned)(hit >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hit, 0));
                float x = z[i];
                asm volatile("" : "+v"(x));  // (its key is made here, for the few, not ahead for all)
                if (x >= limit && place < kCap + KH_MAX_TOP) cand[place] = key_of(x, column_of<THREADS, VEC>(c0, t, i));
                at += __popcll(hit);
              }
            }
          }
        }
        if (tid == 0) count_s[turn ^ 1] = 0;
        __syncthreads();
        n = count_s[turn];
        if (n <= kCap) break;
        __syncthreads();  // (count_s has been read)
        if (tid == 0) count_s[turn] = 0;
        __syncthreads();
      }
      n += have;
      if (n > kCap + have) {
        // (rare: the chunk is read again, from the cache, instead of being kept in registers for this)
        const int end = d.cols - c0 > step ? c0 + step : d.cols;
        // `lo` lets too many through, `hi` too few: the keys between are distinct, so a bound that lets between K and
        // kCap through is found within 64 rounds.  A chunk of at most kCap elements is taken whole.
        key_t lo = 0, hi = ~0ull, found = end - c0 <= kCap ? 0 : hi;
        for (int round = 0; round < 64 && found; ++round) {
          const key_t try_at = lo + (hi - lo) / 2;
          int reach = 0;
          for (int c = c0 + tid; c < end; c += THREADS) reach += key_of(row[c], c) >= try_at;
#pragma unroll
          for (int o = 32; o > 0; o >>= 1) reach += __shfl_xor(reach, o, 64);
          __syncthreads();  // (count_s has been read)
          if (tid == 0) count_s[turn] = 0;
          __syncthreads();
          if (lane == 0) atomicAdd(&count_s[turn], reach);
          __syncthreads();
          const int total = count_s[turn];
          if (total >= K && total <= kCap) {
            found = try_at;
            break;
          }
          if (total > kCap) lo = try_at;
          else hi = try_at;
        }
        __syncthreads();
        if (tid == 0) count_s[turn] = have;
        __syncthreads();
        for (int c = c0 + tid; c < end; c += THREADS) {
          const key_t k = key_of(row[c], c);
          if (k >= found) {
            const int at = atomicAdd(&count_s[turn], 1);
            if (at < kCap + KH_MAX_TOP) cand[at] = k;
          }
        }
        __syncthreads();
        n = min(count_s[turn], kCap + KH_MAX_TOP);
      }
      // a candidate's place is the number of larger ones: four lanes count for one candidate
      for (int i0 = 0; i0 < n; i0 += THREADS / 4) {
        const int i = i0 + (tid >> 2);
        if (i >= n) break;
        const key_t k = cand[i];
        int above = 0;
#pragma unroll 4
        for (int j = tid & 3; j < n; j += 4) above += cand[j] > k;
        above += __shfl_xor(above, 1, 64);
        above += __shfl_xor(above, 2, 64);
        if (above < K && (tid & 3) == 0) best[above] = k;
      }
      have = min(K, n);
      __syncthreads();
    }
    for (int k = tid; k < K; k += THREADS) {
      int c = -1;
      float v = -INFINITY;
      if (k < have) {
        c = (int)~(unsigned)best[k];
        v = row[c];
      }
      idx[(size_t)r * ldidx + k] = c;
      val[(size_t)r * ldval + k] = v;
    }
    if (lse) {
      if (lane == 0) max_s[wave] = m, sum_s[wave] = sum;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < waves; ++w) m = fmaxf(m, max_s[w]);
        const float base = m == -INFINITY ? 0.f : m;
        sum = 0.f;
        for (int w = 0; w < waves; ++w) sum += sum_s[w] * __builtin_amdgcn_exp2f((max_s[w] - base) * 1.44269504088896340736f);
        lse[r] = sum == 0.f ? -INFINITY : base + logf(sum);
      }
    }
    if (r + gridDim.x < d.rows) __syncthreads();  // (the next row may overwrite the shared arrays)
  }
}

// ---- loss and gradient towards a teacher's logits ----------------------------------------------------------------------
struct DistillArgs {
  const float *x;
  MatrixDim d;
  const int32_t *idx; int ldidx;
  const float *val; int ldval;
  int K;
  const int32_t *label;
  const float *weight;
  float T, hard;
  ExpScale soft_scale;
  float *diff; int lddiff;
  float *row_loss;
};

// One workgroup per row.  Every wave has a maximum and sums of its own over its part of the row, so that one barrier joins
// them; the gradient is written from the exponentials in registers, and after a second barrier the few columns that the
// teacher or the label names are written once more with their targets taken off.  The first wave works out the teacher's
// distribution, the last one those columns.  A row of several chunks is read twice.  BOTH: the sums at temperature T and
// at 1 are needed.  4096 rows of 9000 with their gradient: 62.8 us, 4.7 TB/s, three quarters of an
// elementwise pass's rate; the loss alone of 1999 such rows: 18.2 us, 4.0 TB/s, two thirds of a sum's; 70001 columns, read twice by one
// workgroup per row: 1 row 22 us, 64 rows 25, 256 rows 37.  (Rows loaded ahead through LDS as above: 87 and 28 us, fewer waves at a time.)
template <int THREADS, bool VEC, bool BOTH>
__global__ __launch_bounds__(THREADS) void distill_kernel(DistillArgs p) {
  constexpr int waves = THREADS / 64, chunk = THREADS * kHold;
  __shared__ float max_s[waves], sum_t_s[waves], sum_1_s[waves];
  __shared__ int e_col[KH_MAX_TOP];
  __shared__ float e_q[KH_MAX_TOP], e_x[KH_MAX_TOP], e_log[KH_MAX_TOP];
  __shared__ float label_x_s, mass_s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), C = p.d.cols;
  const size_t r = blockIdx.x;
  const float *row = p.x + r * p.d.stride;
  float *out = p.diff ? p.diff + r * p.lddiff : nullptr;
  const float w = p.weight ? p.weight[r] : 1.f;
  const int label = p.hard > 0.f ? p.label[r] : -1;
  const bool labelled = (unsigned)label < (unsigned)C;
  const ExpScale one = {1.44269502f, 1.92596303e-8f};

  // the first wave asks for the teacher's entries (lane k: k and k + 64) before its part of the row
  int col[2] = {-1, -1};
  float v[2] = {-INFINITY, -INFINITY}, x_at[2] = {0.f, 0.f}, label_x = 0.f;
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = lane + 64 * i, c = k < p.K && p.hard < 1.f ? p.idx[r * p.ldidx + k] : -1;
      if ((unsigned)c < (unsigned)C) {
        col[i] = c;
        v[i] = p.val[r * p.ldval + k];
        x_at[i] = row[c];
      }
    }
    if (labelled) label_x = row[label];
  }

  float z[kHold], e1[BOTH ? kHold : 1];
  float m = -INFINITY, sum_t = 0.f, sum_1 = 0.f;
  for (int c0 = 0; c0 < C; c0 += chunk) {
    read_chunk<THREADS, VEC>(row, c0, C, tid, z);
    float most = z[0];
#pragma unroll
    for (int i = 1; i < kHold; ++i) most = fmaxf(most, z[i]);
    most = fmaxf(m, wave_most(most));
    const float base = most == -INFINITY ? 0.f : most;
    float pt = 0.f, p1 = 0.f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const float x = z[i] - base;
      z[i] = exp_scaled(x, p.soft_scale);
      pt += z[i];
      if (BOTH) {
        e1[i] = exp_scaled(x, one);
        p1 += e1[i];
      }
    }
    sum_t = (sum_t == 0.f ? 0.f : sum_t * exp_scaled(m - base, p.soft_scale)) + wave_add(pt);
    if (BOTH) sum_1 = (sum_1 == 0.f ? 0.f : sum_1 * exp_scaled(m - base, one)) + wave_add(p1);
    m = most;
  }
  if (lane == 0) {
    max_s[wave] = m;
    sum_t_s[wave] = sum_t;
    if (BOTH) sum_1_s[wave] = sum_1;
  }
  if (wave == 0) {  // the teacher's distribution
    const float v_max = wave_most(fmaxf(v[0], v[1])), v_base = v_max == -INFINITY ? 0.f : v_max;
    float q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) q[i] = col[i] >= 0 ? exp_scaled(v[i] - v_base, p.soft_scale) : 0.f;
    const float mass = wave_add(q[0] + q[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = lane + 64 * i;
      if (k < p.K) {
        e_col[k] = col[i];
        e_x[k] = x_at[i];
        e_q[k] = mass != 0.f ? q[i] / mass : 0.f;
        e_log[k] = v[i] - v_base;
      }
    }
    if (lane == 0) label_x_s = label_x, mass_s = mass;
  }
  __syncthreads();
  // the row's maximum and sums
  float top = max_s[0];
#pragma unroll
  for (int i = 1; i < waves; ++i) top = fmaxf(top, max_s[i]);
  const float base = top == -INFINITY ? 0.f : top;
  sum_t = sum_1 = 0.f;
#pragma unroll
  for (int i = 0; i < waves; ++i) {
    const float off = max_s[i] == -INFINITY ? 0.f : max_s[i] - base;
    sum_t += sum_t_s[i] * exp_scaled(off, p.soft_scale);
    if (BOTH) sum_1 += sum_1_s[i] * exp_scaled(off, one);
  }
  if (!BOTH) sum_1 = sum_t;  // one of the two parts is absent, or T = 1
  const float mass = mass_s;
  const bool some = mass != 0.f;  // (true for NaN)
  const bool nothing = w == 0.f || (top == -INFINITY && sum_t == 0.f);  // to learn from this row
  const float ws = w * (1.f - p.hard) * p.T, wh = w * p.hard;
  const float ft = nothing || !some ? 0.f : ws / sum_t, f1 = nothing || !labelled ? 0.f : wh / sum_1;

  if (out) {
    const bool single = C <= chunk;
    // (of a single chunk: the exponentials in the registers are relative to the wave's own maximum.  A wave whose columns are
    // all -inf has none and holds zeros: 0 - base would overflow where the row lies far below 0, and 0 * inf is NaN)
    const float off = m == -INFINITY ? 0.f : m - base;
    const float st = (BOTH ? ft : ft + f1) * exp_scaled(off, p.soft_scale);
    const float s1 = BOTH ? f1 * exp_scaled(off, one) : 0.f;
    for (int c0 = 0; c0 < C; c0 += chunk) {
      if (single) {
#pragma unroll
        for (int i = 0; i < kHold; ++i) z[i] = BOTH ? __builtin_fmaf(st, z[i], s1 * e1[i]) : st * z[i];
      } else {
        read_chunk<THREADS, VEC>(row, c0, C, tid, z);
#pragma unroll
        for (int i = 0; i < kHold; ++i) {
          const float x = z[i] - base;
          z[i] = BOTH ? __builtin_fmaf(ft, exp_scaled(x, p.soft_scale), f1 * exp_scaled(x, one)) : (ft + f1) * exp_scaled(x, p.soft_scale);
        }
      }
      if (nothing) {  // (whatever the row holds)
#pragma unroll
        for (int i = 0; i < kHold; ++i) z[i] = 0.f;
      }
      constexpr int n = VEC ? 4 : 1;
#pragma unroll
      for (int i = 0; i < kHold; i += n) {
        const int c = column_of<THREADS, VEC>(c0, tid, i);
        if (VEC && c + 4 <= C) {
          *reinterpret_cast<v4f *>(out + c) = (v4f){z[i], z[(i + 1) % kHold], z[(i + 2) % kHold], z[(i + 3) % kHold]};
        } else {
#pragma unroll
          for (int j = 0; j < n; ++j)
            if (c + j < C) out[c + j] = z[i + j];
        }
      }
    }
    __syncthreads();  // the plain values are written: now the columns with a target, each from its own x
    if (wave == waves - 1 && !nothing) {
      bool named = false;  // the label, by an entry
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = lane + 64 * i, c = k < p.K ? e_col[k] : -1;
        named |= __ballot(c >= 0 && c == label) != 0;
        float q = 0.f;
        for (int j = 0; j < p.K; ++j) q += e_col[j] == c ? e_q[j] : 0.f;
        if (c >= 0) {
          const float x = e_x[k] - base;
          float g = BOTH ? __builtin_fmaf(ft, exp_scaled(x, p.soft_scale), f1 * exp_scaled(x, one)) : (ft + f1) * exp_scaled(x, p.soft_scale);
          g -= ws * q;
          if (labelled && c == label) g -= wh;
          out[c] = g;
        }
      }
      if (labelled && !named && lane == 0) {
        const float x = label_x_s - base;
        const float g = BOTH ? __builtin_fmaf(ft, exp_scaled(x, p.soft_scale), f1 * exp_scaled(x, one)) : (ft + f1) * exp_scaled(x, p.soft_scale);
        out[label] = g - wh;
      }
    }
  }
  if (p.row_loss && wave == 0) {
    double soft = 0.0;
    if (some && !nothing) {
      const double logs = log((double)sum_t) - log((double)mass);
      for (int k = lane; k < p.K; k += 64) {
        const float q = e_q[k];
        if (q != 0.f) soft += (double)q * (((double)e_log[k] - ((double)e_x[k] - (double)top)) / (double)p.T + logs);
      }
      soft = kh::wave_sum_d(soft);
    }
    if (lane == 0) {
      double loss = (1.0 - (double)p.hard) * (double)p.T * (double)p.T * soft;
      if (labelled) loss += (double)p.hard * (log((double)sum_1) - ((double)label_x_s - (double)top));
      p.row_loss[r] = nothing ? 0.f : (float)((double)w * loss);
    }
  }
}

// One workgroup behind the rows' (256 rows 1.8 us, 4096 rows 3 to 4, 2^25 rows 47 ms).
// loss[0] += the rows' losses, in a fixed order: thread t adds rows t, t + 256, ..., then the threads' sums in a tree
__global__ __launch_bounds__(256) void sum_rows_kernel(const float *row_loss, int rows, double *loss) {
  __shared__ double sd[4];
  double t = 0.0;
  for (unsigned i = threadIdx.x; i < (unsigned)rows; i += 256) t += (double)row_loss[i];  // (past 2^31 an int would wrap around)
  t = kh::wave_sum_d(t);
  if ((threadIdx.x & 63) == 0) sd[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) loss[0] += sd[0] + sd[1] + sd[2] + sd[3];
}

// the library works on the device that hipK_init chose
int check_device() {
  int now = -1;
  KH_HIP(hipGetDevice(&now));
  KH_REQUIRE(now == kh::ctx().device);
  return KH_OK;
}

template <int THREADS, bool VEC, bool AHEAD>
void launch_row_top_as(hipStream_t st, const float *mat, MatrixDim d, int K, int32_t *idx, int ldidx, float *val, int ldval,
                       float *lse) {
  // as many workgroups as run at once, each with its share of the rows
  constexpr unsigned by_lds = 163840u / (THREADS * kHold * 4u + (kCap + 2 * KH_MAX_TOP) * 8u + 2048u);
  const unsigned rows = (unsigned)d.rows, most = 256u * by_lds;
  if constexpr (AHEAD) row_top_kernel<THREADS, VEC, true><<<rows < most ? rows : most, THREADS, 0, st>>>(mat, d, K, idx, ldidx, val, ldval, lse);
  else row_top_kernel<THREADS, VEC, false><<<rows, THREADS, 0, st>>>(mat, d, K, idx, ldidx, val, ldval, lse);
}
// A grid counts its threads in 32 bits: more rows than this go in several launches.
constexpr int kRowsAtOnce = 1 << 21;
template <bool VEC>
void launch_row_top(hipStream_t st, const float *mat, MatrixDim d, int K, int32_t *idx, int ldidx, float *val, int ldval,
                    float *lse) {
  // the fewest threads that hold the row
  if (d.cols <= 64 * kHold && K <= 64) launch_row_top_as<64, VEC, false>(st, mat, d, K, idx, ldidx, val, ldval, lse);
  else if (d.cols <= 256 * kHold) launch_row_top_as<256, VEC, false>(st, mat, d, K, idx, ldidx, val, ldval, lse);
  else if (d.cols <= 512 * kHold) launch_row_top_as<512, VEC, false>(st, mat, d, K, idx, ldidx, val, ldval, lse);
  else launch_row_top_as<1024, VEC, true>(st, mat, d, K, idx, ldidx, val, ldval, lse);
}

template <bool VEC, bool BOTH>
void launch_distill(hipStream_t st, const DistillArgs &p) {
  const unsigned rows = (unsigned)p.d.rows;
  if (p.d.cols <= 64 * kHold) distill_kernel<64, VEC, BOTH><<<rows, 64, 0, st>>>(p);
  else if (p.d.cols <= 256 * kHold) distill_kernel<256, VEC, BOTH><<<rows, 256, 0, st>>>(p);
  else if (p.d.cols <= 512 * kHold) distill_kernel<512, VEC, BOTH><<<rows, 512, 0, st>>>(p);
  else distill_kernel<1024, VEC, BOTH><<<rows, 1024, 0, st>>>(p);
}

int too_large(const char *what, int K) {
  snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "%s: K = %d, at most %d", what, K, KH_MAX_TOP);
  return KH_ERR_TOO_LARGE;
}

constexpr int kMaxCols = 1 << 30;  // columns are counted in 32 bits, a chunk further than the row goes
int too_wide(int cols) {
  snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "%d columns: at most %d", cols, kMaxCols);
  return KH_ERR_TOO_LARGE;
}

}  // namespace

KH_EXPORT int hipF_row_top(khStream_t s, const float *mat, MatrixDim d, int32_t K, int32_t *idx, int32_t ldidx, float *val,
                           int32_t ldval, float *lse) {
  KH_REQUIRE(kh::dim_ok(d) && K >= 1 && ldidx >= K && ldval >= K);
  if (K > KH_MAX_TOP) return too_large(__func__, K);
  if (d.cols > kMaxCols) return too_wide(d.cols);
  KH_REQUIRE(d.rows == 0 || (idx != nullptr && val != nullptr && (d.cols == 0 || mat != nullptr)));
  int rc = kh::check_apart(__func__, {{"idx", idx, d.rows, K, ldidx}, {"val", val, d.rows, K, ldval}, {"lse", lse, 1, d.rows, d.rows}},
                           {{"mat", mat, d.rows, d.cols, d.stride}});
  if (rc != KH_OK) return rc;
  KH_CHECK_INIT();
  rc = check_device();
  if (rc != KH_OK) return rc;
  if (d.rows == 0) return KH_OK;
  hipStream_t st = kh::pick(s);
  const bool vec = kh::aligned16(mat) && d.stride % 4 == 0;
  for (size_t r = 0; r < (size_t)d.rows; r += kRowsAtOnce) {
    const MatrixDim part = {std::min(d.rows - (int)r, kRowsAtOnce), d.cols, d.stride};
    float *l = lse ? lse + r : nullptr;
    if (vec) launch_row_top<true>(st, mat + r * d.stride, part, K, idx + r * ldidx, ldidx, val + r * ldval, ldval, l);
    else launch_row_top<false>(st, mat + r * d.stride, part, K, idx + r * ldidx, ldidx, val + r * ldval, ldval, l);
    rc = kh::launch_status();
    if (rc != KH_OK) return rc;
  }
  return KH_OK;
}

KH_EXPORT int hipF_distill_eval(khStream_t s, const float *x, MatrixDim d, const int32_t *idx, int32_t ldidx,
                                const float *val, int32_t ldval, int32_t K, const int32_t *label, const float *weight,
                                float temperature, float hard_weight, float *diff, int32_t lddiff, float *row_loss,
                                double *loss) {
  KH_REQUIRE(kh::dim_ok(d) && K >= 1 && ldidx >= K && ldval >= K);
  if (K > KH_MAX_TOP) return too_large(__func__, K);
  if (d.cols > kMaxCols) return too_wide(d.cols);
  // (the smallest normal float: log2(e) / T is a float then, and 0 / T a number)
  KH_REQUIRE(temperature >= 1.17549435e-38f && temperature <= 3.402823466e38f);
  KH_REQUIRE(hard_weight >= 0.f && hard_weight <= 1.f);
  KH_REQUIRE(d.rows == 0 || (idx != nullptr && val != nullptr && (d.cols == 0 || x != nullptr)));
  KH_REQUIRE(d.rows == 0 || hard_weight == 0.f || label != nullptr);
  KH_REQUIRE(diff == nullptr || lddiff >= d.cols);
  KH_REQUIRE(diff != x || lddiff == d.stride);
  KH_REQUIRE(loss == nullptr || d.rows == 0 || row_loss != nullptr);
  // (diff may be x itself; the table is not read where only hard labels count, labels not where they do not)
  const int table_rows = hard_weight < 1.f ? d.rows : 0;
  int rc = kh::check_apart(__func__,
                           {{"diff", diff, d.rows, d.cols, lddiff}, {"row_loss", row_loss, 1, d.rows, d.rows}, {"loss", loss, d.rows > 0, 2, 2}},
                           {{"x", diff == x ? nullptr : x, d.rows, d.cols, d.stride}, {"idx", idx, table_rows, K, ldidx},
                            {"val", val, table_rows, K, ldval}, {"label", label, hard_weight > 0.f, d.rows, d.rows},
                            {"weight", weight, 1, d.rows, d.rows}});
  // (with diff in the place of x, what overlaps x overlaps diff)
  if (rc != KH_OK) return rc;
  KH_CHECK_INIT();
  rc = check_device();
  if (rc != KH_OK) return rc;
  if (d.rows == 0) return KH_OK;
  hipStream_t st = kh::pick(s);
  const bool vec = kh::aligned16(x) && d.stride % 4 == 0 && (diff == nullptr || (kh::aligned16(diff) && lddiff % 4 == 0));
  const bool both = hard_weight > 0.f && hard_weight < 1.f && temperature != 1.f;
  for (size_t r = 0; r < (size_t)d.rows; r += kRowsAtOnce) {
    const MatrixDim part = {std::min(d.rows - (int)r, kRowsAtOnce), d.cols, d.stride};
    const DistillArgs p = {x + r * d.stride, part, idx + r * ldidx, ldidx, val + r * ldval, ldval, K, label ? label + r : nullptr,
                           weight ? weight + r : nullptr, temperature, hard_weight,
                           exp_scale(hard_weight == 1.f ? 1.0 : 1.0 / (double)temperature), diff ? diff + r * lddiff : nullptr, lddiff,
                           row_loss ? row_loss + r : nullptr};
    if (vec && both) launch_distill<true, true>(st, p);
    else if (vec) launch_distill<true, false>(st, p);
    else if (both) launch_distill<false, true>(st, p);
    else launch_distill<false, false>(st, p);
    rc = kh::launch_status();
    if (rc != KH_OK) return rc;
  }
  if (loss == nullptr) return KH_OK;
  sum_rows_kernel<<<1, 256, 0, st>>>(row_loss, d.rows, loss);
  return kh::launch_status();
}
