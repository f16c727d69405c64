// Learning from another network's outputs: hipF_row_top (a row's largest logits) and hipF_distill_eval (loss and gradient
// towards them, mixed with hard labels); include/kaldi_hip.h has the formulas.
//
// Both are bound by reading (and writing) the logits once.  One workgroup takes one row; its threads hold up to kHold
// floats of it each, so a row of up to 1024 * kHold = 20480 columns stays in registers between the maximum, the sum and the
// output.  A longer row is gone through in such chunks.
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
template <int THREADS, bool VEC>
__device__ __forceinline__ void load_chunk(const float *row, int c0, int C, int tid, float (&z)[kHold]) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < kHold; i += 4) {
      const int c = column_of<THREADS, VEC>(c0, tid, i);
      if (c + 4 <= C) {
        const v4f v = *reinterpret_cast<const v4f *>(row + c);
        z[i] = v.x, z[i + 1] = v.y, z[i + 2] = v.z, z[i + 3] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) z[i + j] = c + j < C ? row[c + j] : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int c = column_of<THREADS, VEC>(c0, tid, i);
      z[i] = c < C ? row[c] : -INFINITY;
    }
  }
}

template <int THREADS>
__device__ __forceinline__ float all_sum(float v, float *red) {
  if (THREADS == 64) return kh::wave_sum(v);
  return kh::block_sum(v, red);
}
// (fmaxf passes over NaN: a NaN shows up in the sums)
template <int THREADS>
__device__ __forceinline__ float all_max(float v, float *red) {
  if (THREADS == 64) return kh::wave_max(v);
  return kh::block_max(v, red);
}

// ---- the K largest of a row -------------------------------------------------------------------------------------------
// Order of the answer: by value, NaN above everything, -0 = +0, then by ascending column.  A 64-bit key has it: the
// float's bits made monotone in the upper half, the complement of the column in the lower.
typedef unsigned long long key_t;
__device__ __forceinline__ unsigned ordered(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned b = __float_as_uint(x + 0.f);  // -0 + 0 = +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ key_t key_of(float x, int c) { return (key_t)ordered(x) << 32 | (unsigned)~c; }

constexpr int kCap = 1024;  // candidates of a chunk, next to the KH_MAX_TOP of the chunks before

// One workgroup per row, chunk by chunk.  A chunk's threads form G >= K groups; the K-th largest of the groups' maxima is
// a lower bound of the chunk's K-th largest, which leaves few more than K candidates where large values are spread over
// the row.  Candidates (also above the K-th of the chunks before) are collected in LDS and ranked by counting; the K
// largest are kept.  Where more than kCap pass (large values crowded into few groups) the bound is raised by bisection
// on the keys, which are distinct.
template <int THREADS, bool VEC>
__global__ __launch_bounds__(THREADS) void row_top_kernel(const float *mat, MatrixDim d, int K, int32_t *idx, int ldidx,
                                                          float *val, int ldval, float *lse) {
  constexpr int G = THREADS < 256 ? THREADS : 256;  // groups: one per thread, or 256
  __shared__ key_t cand[kCap + KH_MAX_TOP];
  __shared__ key_t best[KH_MAX_TOP];
  __shared__ key_t gmax[G];
  __shared__ key_t bound_s;
  __shared__ int count_s;
  __shared__ float red[16];
  const int tid = threadIdx.x;
  const float *row = mat + (size_t)blockIdx.x * d.stride;
  int have = 0;         // valid entries of best[]
  float m = -INFINITY;  // running maximum and sum of exp(x - m)
  float sum = 0.f;
  const ExpScale one = {1.44269502f, 1.92596303e-8f};

  for (int c0 = 0; c0 < d.cols; c0 += THREADS * kHold) {
    float z[kHold];
    load_chunk<THREADS, VEC>(row, c0, d.cols, tid, z);
    if (lse) {
      float cm = z[0];
#pragma unroll
      for (int i = 1; i < kHold; ++i) cm = fmaxf(cm, z[i]);
      cm = fmaxf(m, all_max<THREADS>(cm, red));
      // (a NaN in a chunk of -inf: m stays -inf, and the sum takes the NaN)
      const float base = cm == -INFINITY ? 0.f : cm;
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < kHold; ++i) part += exp_scaled(z[i] - base, one);
      part = all_sum<THREADS>(part, red);
      sum = (sum == 0.f ? 0.f : sum * expf(m - base)) + part;
      m = cm;
    }
    // the thread's largest, then the group's
    key_t mine = 0;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int c = column_of<THREADS, VEC>(c0, tid, i);
      const key_t k = key_of(z[i], c);
      if (c < d.cols && k > mine) mine = k;
    }
    constexpr int per = THREADS / G;
#pragma unroll
    for (int o = per / 2; o > 0; o >>= 1) {
      const key_t other = __shfl_xor(mine, o, 64);
      mine = other > mine ? other : mine;
    }
    __syncthreads();  // (the chunk before is done with the shared arrays)
    if (tid % per == 0) gmax[tid / per] = mine;
    if (tid == 0) {
      count_s = 0;
      bound_s = have == K ? best[K - 1] : 0;
    }
    __syncthreads();
    // The K-th largest of the groups' maxima, by counting; empty groups hold 0, which bounds nothing.  K > G (64
    // threads): no bound from here.
    if (tid < G && K <= G) {
      const key_t k = gmax[tid];
      int above = 0;
      for (int j = 0; j < G; ++j) above += gmax[j] > k;
      if (above == K - 1 && k > bound_s) bound_s = k;  // keys are distinct but for 0: one thread writes, or all a 0
    }
    __syncthreads();
    // Candidates: this chunk's keys from the bound on.  `lo` lets too many through or is the answer, `hi` too few; keys are
    // distinct, so the two cannot meet with more than kCap >= K + 1 between them: at most 64 rounds.
    key_t lo = bound_s, hi = ~0ull, try_at = lo;
    for (int round = 0; round <= 64; ++round) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int c = column_of<THREADS, VEC>(c0, tid, i);
        n += c < d.cols && key_of(z[i], c) >= try_at;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
      __syncthreads();  // (count_s of the round before has been read)
      if (tid == 0) count_s = 0;
      __syncthreads();
      if ((tid & 63) == 0) atomicAdd(&count_s, n);
      __syncthreads();
      const int total = count_s;
      if (total <= kCap && (round == 0 || total >= K)) {
        lo = try_at;
        break;
      }
      if (total > kCap) lo = try_at;
      else hi = try_at;
      try_at = lo + (hi - lo) / 2;
    }
    __syncthreads();
    if (tid == 0) count_s = have;
    if (tid < have) cand[tid] = best[tid];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int c = column_of<THREADS, VEC>(c0, tid, i);
      const key_t k = key_of(z[i], c);
      if (c < d.cols && k >= lo) {
        const int at = atomicAdd(&count_s, 1);
        if (at < kCap + KH_MAX_TOP) cand[at] = k;
      }
    }
    __syncthreads();
    const int n = min(count_s, kCap + KH_MAX_TOP);
    for (int i = tid; i < n; i += THREADS) {
      const key_t k = cand[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += cand[j] > k;
      if (above < K) best[above] = k;
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
    idx[(size_t)blockIdx.x * ldidx + k] = c;
    val[(size_t)blockIdx.x * ldval + k] = v;
  }
  if (lse && tid == 0) lse[blockIdx.x] = sum == 0.f ? -INFINITY : (float)((double)m + log((double)sum));
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
  float T, inv_t, hard;
  ExpScale soft_scale;
  float *diff; int lddiff;
  float *row_loss;
};

// One workgroup per row.  The teacher's entries sit in LDS; the row's maximum and sums are taken from registers, the
// gradient is written from them, and the few columns that the teacher or the label names are written once more with
// their targets taken off, after a barrier.  BOTH: the sums at temperature T and at 1 are needed.
template <int THREADS, bool VEC, bool BOTH>
__global__ __launch_bounds__(THREADS) void distill_kernel(DistillArgs p) {
  __shared__ float red[16];
  __shared__ int e_col[KH_MAX_TOP];
  __shared__ float e_val[KH_MAX_TOP], e_q[KH_MAX_TOP], e_x[KH_MAX_TOP];
  __shared__ double e_loss[KH_MAX_TOP];
  const int tid = threadIdx.x, r = blockIdx.x, C = p.d.cols;
  const float *row = p.x + (size_t)r * p.d.stride;
  float *out = p.diff ? p.diff + (size_t)r * p.lddiff : nullptr;
  const float w = p.weight ? p.weight[r] : 1.f;
  const int label = p.hard > 0.f ? p.label[r] : -1;
  const bool labelled = (unsigned)label < (unsigned)C;
  const ExpScale one = {1.44269502f, 1.92596303e-8f};

  for (int k = tid; k < p.K; k += THREADS) {
    const int c = p.hard < 1.f ? p.idx[(size_t)r * p.ldidx + k] : -1;
    const bool there = (unsigned)c < (unsigned)C;
    e_col[k] = there ? c : -1;
    e_val[k] = there ? p.val[(size_t)r * p.ldval + k] : -INFINITY;
    e_x[k] = there ? row[c] : 0.f;
  }
  const float label_x = labelled ? row[label] : 0.f;

  // the row's maximum and sums
  float z[kHold];
  float m = -INFINITY, sum_t = 0.f, sum_1 = 0.f;
  const bool single = C <= THREADS * kHold;
  for (int c0 = 0; c0 < C; c0 += THREADS * kHold) {
    load_chunk<THREADS, VEC>(row, c0, C, tid, z);
    float cm = z[0];
#pragma unroll
    for (int i = 1; i < kHold; ++i) cm = fmaxf(cm, z[i]);
    cm = fmaxf(m, all_max<THREADS>(cm, red));
    const float base = cm == -INFINITY ? 0.f : cm;
    float pt = 0.f, p1 = 0.f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      pt += exp_scaled(z[i] - base, p.soft_scale);
      if (BOTH) p1 += exp_scaled(z[i] - base, one);
    }
    const float at = all_sum<THREADS>(pt, red), a1 = BOTH ? all_sum<THREADS>(p1, red) : 0.f;
    sum_t = (sum_t == 0.f ? 0.f : sum_t * exp_scaled(m - base, p.soft_scale)) + at;
    if (BOTH) sum_1 = (sum_1 == 0.f ? 0.f : sum_1 * exp_scaled(m - base, one)) + a1;
    m = cm;
  }
  if (!BOTH) sum_1 = sum_t;  // one of the two parts is absent, or T = 1
  __syncthreads();           // (the entries are in LDS, and every x of the row that the scatter needs has been read)

  if (w == 0.f || (m == -INFINITY && sum_t == 0.f)) {  // nothing to learn from this row
    if (out)
      for (int c = tid; c < C; c += THREADS) out[c] = 0.f;
    if (p.row_loss && tid == 0) p.row_loss[r] = 0.f;
    return;
  }

  // the teacher's distribution
  float vm = -INFINITY;
  for (int k = 0; k < p.K; ++k) vm = fmaxf(vm, e_val[k]);
  float vsum = 0.f;
  for (int k = 0; k < p.K; ++k)
    if (e_col[k] >= 0) vsum += exp_scaled(e_val[k] - (vm == -INFINITY ? 0.f : vm), p.soft_scale);
  const bool some = vsum != 0.f;  // (true for NaN)
  for (int k = tid; k < p.K; k += THREADS) {
    float q = 0.f;
    double part = 0.0;
    if (e_col[k] >= 0 && some) {
      q = exp_scaled(e_val[k] - (vm == -INFINITY ? 0.f : vm), p.soft_scale) / vsum;
      if (q != 0.f) {
        const double logq = ((double)e_val[k] - (double)vm) / (double)p.T - log((double)vsum);
        const double logp = ((double)e_x[k] - (double)m) / (double)p.T - log((double)sum_t);
        part = (double)q * (logq - logp);
      }
    }
    e_q[k] = q;
    e_loss[k] = part;
  }
  __syncthreads();
  if (p.row_loss && tid == 0) {
    double soft = 0.0;
    for (int k = 0; k < p.K; ++k) soft += e_loss[k];
    double loss = (1.0 - (double)p.hard) * (double)p.T * (double)p.T * soft;
    if (labelled) loss += (double)p.hard * (log((double)sum_1) - ((double)label_x - (double)m));
    p.row_loss[r] = (float)((double)w * loss);
  }
  if (!out) return;

  const float ws = w * (1.f - p.hard) * p.T, wh = w * p.hard;
  const float ft = some ? ws / sum_t : 0.f, f1 = labelled ? wh / sum_1 : 0.f;
  const float base = m == -INFINITY ? 0.f : m;
  for (int c0 = 0; c0 < C; c0 += THREADS * kHold) {
    if (!single) load_chunk<THREADS, VEC>(row, c0, C, tid, z);
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const float x = z[i] - base;
      z[i] = BOTH ? __builtin_fmaf(ft, exp_scaled(x, p.soft_scale), f1 * exp_scaled(x, one)) : (ft + f1) * exp_scaled(x, p.soft_scale);
    }
    if (VEC) {
#pragma unroll
      for (int i = 0; i < kHold; i += 4) {
        const int c = column_of<THREADS, VEC>(c0, tid, i);
        if (c + 4 <= C) *reinterpret_cast<v4f *>(out + c) = (v4f){z[i], z[i + 1], z[i + 2], z[i + 3]};
        else
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < C) out[c + j] = z[i + j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int c = column_of<THREADS, VEC>(c0, tid, i);
        if (c < C) out[c] = z[i];
      }
    }
  }
  __syncthreads();  // the plain values are written: now the columns with a target, each from its own x
  bool label_done = !labelled;
  for (int k = 0; k < p.K; ++k) label_done |= e_col[k] == label;
  for (int k = tid; k <= p.K; k += THREADS) {
    const bool entry = k < p.K;
    if (entry ? e_col[k] < 0 : label_done) continue;
    const int c = entry ? e_col[k] : label;
    float q = 0.f;
    for (int j = 0; j < p.K; ++j) q += e_col[j] == c ? e_q[j] : 0.f;
    const float x = (entry ? e_x[k] : label_x) - base;
    float g = BOTH ? __builtin_fmaf(ft, exp_scaled(x, p.soft_scale), f1 * exp_scaled(x, one)) : (ft + f1) * exp_scaled(x, p.soft_scale);
    g -= ws * q;
    if (labelled && c == label) g -= wh;
    out[c] = g;
  }
}

// loss[0] += the rows' losses, in a fixed order
__global__ __launch_bounds__(256) void sum_rows_kernel(const float *row_loss, int rows, double *loss) {
  __shared__ double sd[4];
  double t = 0.0;
  for (int i = threadIdx.x; i < rows; i += 256) t += (double)row_loss[i];
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

template <bool VEC>
void launch_row_top(hipStream_t st, const float *mat, MatrixDim d, int K, int32_t *idx, int ldidx, float *val, int ldval,
                    float *lse) {
  const unsigned rows = (unsigned)d.rows;
  // the fewest threads that hold the row; K candidates need K groups
  if (d.cols <= 64 * kHold && K <= 64)
    row_top_kernel<64, VEC><<<rows, 64, 0, st>>>(mat, d, K, idx, ldidx, val, ldval, lse);
  else if (d.cols <= 256 * kHold)
    row_top_kernel<256, VEC><<<rows, 256, 0, st>>>(mat, d, K, idx, ldidx, val, ldval, lse);
  else if (d.cols <= 512 * kHold)
    row_top_kernel<512, VEC><<<rows, 512, 0, st>>>(mat, d, K, idx, ldidx, val, ldval, lse);
  else
    row_top_kernel<1024, VEC><<<rows, 1024, 0, st>>>(mat, d, K, idx, ldidx, val, ldval, lse);
}

template <bool VEC, bool BOTH>
void launch_distill(hipStream_t st, const DistillArgs &p) {
  const unsigned rows = (unsigned)p.d.rows;
  if (p.d.cols <= 256 * kHold) distill_kernel<256, VEC, BOTH><<<rows, 256, 0, st>>>(p);
  else if (p.d.cols <= 512 * kHold) distill_kernel<512, VEC, BOTH><<<rows, 512, 0, st>>>(p);
  else distill_kernel<1024, VEC, BOTH><<<rows, 1024, 0, st>>>(p);
}

int too_large(const char *what, int K) {
  snprintf(kh::ctx().last_msg, sizeof(kh::ctx().last_msg), "%s: K = %d, at most %d", what, K, KH_MAX_TOP);
  return KH_ERR_TOO_LARGE;
}

}  // namespace

KH_EXPORT int hipF_row_top(khStream_t s, const float *mat, MatrixDim d, int32_t K, int32_t *idx, int32_t ldidx, float *val,
                           int32_t ldval, float *lse) {
  KH_REQUIRE(kh::dim_ok(d) && K >= 1 && ldidx >= K && ldval >= K);
  if (K > KH_MAX_TOP) return too_large(__func__, K);
  KH_REQUIRE(d.rows == 0 || (idx != nullptr && val != nullptr && (d.cols == 0 || mat != nullptr)));
  KH_CHECK_INIT();
  int rc = check_device();
  if (rc != KH_OK) return rc;
  if (d.rows == 0) return KH_OK;
  hipStream_t st = kh::pick(s);
  if (kh::aligned16(mat) && d.stride % 4 == 0) launch_row_top<true>(st, mat, d, K, idx, ldidx, val, ldval, lse);
  else launch_row_top<false>(st, mat, d, K, idx, ldidx, val, ldval, lse);
  return kh::launch_status();
}

KH_EXPORT int hipF_distill_eval(khStream_t s, const float *x, MatrixDim d, const int32_t *idx, int32_t ldidx,
                                const float *val, int32_t ldval, int32_t K, const int32_t *label, const float *weight,
                                float temperature, float hard_weight, float *diff, int32_t lddiff, float *row_loss,
                                double *loss) {
  KH_REQUIRE(kh::dim_ok(d) && K >= 1 && ldidx >= K && ldval >= K);
  if (K > KH_MAX_TOP) return too_large(__func__, K);
  KH_REQUIRE(temperature > 0.f && temperature <= 3.402823466e38f);
  KH_REQUIRE(hard_weight >= 0.f && hard_weight <= 1.f);
  KH_REQUIRE(d.rows == 0 || (idx != nullptr && val != nullptr && (d.cols == 0 || x != nullptr)));
  KH_REQUIRE(d.rows == 0 || hard_weight == 0.f || label != nullptr);
  KH_REQUIRE(diff == nullptr || lddiff >= d.cols);
  KH_REQUIRE(diff != x || lddiff == d.stride);
  KH_REQUIRE(loss == nullptr || d.rows == 0 || row_loss != nullptr);
  KH_CHECK_INIT();
  int rc = check_device();
  if (rc != KH_OK) return rc;
  if (d.rows == 0) return KH_OK;
  hipStream_t st = kh::pick(s);
  DistillArgs p = {x, d, idx, ldidx, val, ldval, K, label, weight, temperature, 1.f / temperature, hard_weight,
                   exp_scale(hard_weight == 1.f ? 1.0 : 1.0 / (double)temperature), diff, lddiff, row_loss};
  const bool vec = kh::aligned16(x) && d.stride % 4 == 0 && (diff == nullptr || (kh::aligned16(diff) && lddiff % 4 == 0));
  const bool both = hard_weight > 0.f && hard_weight < 1.f && temperature != 1.f;
  if (vec && both) launch_distill<true, true>(st, p);
  else if (vec) launch_distill<true, false>(st, p);
  else if (both) launch_distill<false, true>(st, p);
  else launch_distill<false, false>(st, p);
  rc = kh::launch_status();
  if (rc != KH_OK || loss == nullptr) return rc;
  sum_rows_kernel<<<1, 256, 0, st>>>(row_loss, d.rows, loss);
  return kh::launch_status();
}
