// Kernels around the head's GEMMs for losses on log-probabilities: packing the
// rows that count, joining the row statistics, the teacher's entries and the
// per-row part of the distillation loss, and bringing gradients back to the
// batch's order.
//
// Rows that a mask or ignore_index leaves out (prompts, padding: a third of the
// rows of a preference batch) are taken out before the GEMMs: the rows that
// count move to the front of a copy of e, in order, and every GEMM runs on
// those alone.  The copy moves 4 N D bytes (10 us at N = D = 4096) where the
// GEMMs cost 3 us per row saved there.
//
// Distillation of a row with logits z (already divided by the temperature) and
// teacher entries S with probabilities p_v (P their sum, r what they leave over):
//     L = sum_S p_v (log p_v - log q_v) + r (log r - log q_r),  q_r = 1 - sum_S q_v
//     dL/dz_v = (P + r) q_v - p_v                  for v in S
//             = e^(z_v - lse_r) ((P + r) q_r - r)  for the others
// lse_r, the log-sum-exp over the columns outside of S, is summed directly
// (never as 1 - sum), so a tail of 1e-6 keeps its digits; the others'
// gradient has one coefficient per row, and S is a list of K values per row.
#include <type_traits>

#include "kernels.cuh"

namespace cce {
namespace {

// ---------------------------------------------------------------------------
// packing
// ---------------------------------------------------------------------------

constexpr int kPackThreads = 1024;
constexpr int kPackPer = 8;

// One block walks the rows in order: a scan of the counting rows gives each its
// place, so the packed order is the batch's and does not depend on scheduling.
template <typename TT>  // target type; void: rows count by `mask` alone
__global__ void __launch_bounds__(kPackThreads)
rows_pack_kernel(const TT* __restrict__ targets, int64_t ignore_index, int has_ignore,
                 const uint8_t* __restrict__ mask, int64_t N, const RowsView R, uint8_t* __restrict__ mask_out,
                 float* __restrict__ per_row_out, float* __restrict__ tgt, uint32_t* __restrict__ words) {
  __shared__ int warp_tot[32];
  __shared__ int base_sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) base_sh = 0;
  if (words && threadIdx.x < 2) words[threadIdx.x] = 0u;
  __syncthreads();
  for (int64_t r0 = 0; r0 < N; r0 += kPackThreads * kPackPer) {
    const int64_t n0 = r0 + (int64_t)threadIdx.x * kPackPer;
    int32_t t[kPackPer];
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < kPackPer; ++j) {
      t[j] = 0;
      if (n0 + j < N) {
        bool ok = mask == nullptr || mask[n0 + j] != 0;
        if constexpr (!std::is_void<TT>::value) {
          const int64_t x = (int64_t)targets[n0 + j];
          ok = ok && !(has_ignore && x == ignore_index);
          t[j] = (int32_t)(x < INT32_MIN ? INT32_MIN : x > INT32_MAX ? INT32_MAX : x);
        }
        if (ok) bits |= 1u << j;
      }
    }
    const int cnt = __popc(bits);
    int incl = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int w = warp_tot[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      warp_tot[lane] = w;
    }
    __syncthreads();
    int at = base_sh + incl - cnt + (warp > 0 ? warp_tot[warp - 1] : 0);
#pragma unroll
    for (int j = 0; j < kPackPer; ++j) {
      if (n0 + j < N) {
        const bool ok = (bits >> j) & 1u;
        R.pos[n0 + j] = ok ? at : -1;
        if (mask_out) mask_out[n0 + j] = ok ? 1 : 0;
        if (ok) {
          R.row_of[at] = (int32_t)(n0 + j);
          if constexpr (!std::is_void<TT>::value) {
            R.targets[at] = t[j];
            tgt[at] = 0.f;  // (stays for a target that is no column)
          }
          ++at;
        } else if (per_row_out) {
          per_row_out[n0 + j] = 0.f;
        }
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) base_sh += warp_tot[31];
    __syncthreads();
  }
  if (threadIdx.x == 0) *R.count = base_sh;
}

// A warp per row of 16-bit values: dst[i] = src[row_of[i]], zeros behind the
// count (the grad_c GEMM multiplies those rows by zeros, so they must be
// numbers), or with no list dst[i] = src[i]; columns behind `cols` are zeros.
// kMax: float16, the largest finite |value| as its bits into *word.
template <bool kVec, bool kMax>
__global__ void __launch_bounds__(256)
rows_copy_kernel(const uint16_t* __restrict__ src, int64_t rows, int64_t cols, int64_t src_ld,
                 const int32_t* __restrict__ row_of, const int32_t* __restrict__ count, uint16_t* __restrict__ dst,
                 int64_t dst_ld, uint32_t* __restrict__ word) {
  const int lane = threadIdx.x & 31;
  uint32_t m = 0;
  auto larger = [&](uint32_t x) {
    x &= 0x7fffu;
    m = max(m, x < 0x7c00u ? x : 0u);
  };
  const int64_t live = count ? *count : rows;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows; i += (int64_t)gridDim.x * 8) {
    const uint16_t* p = i < live ? src + (row_of ? row_of[i] : i) * src_ld : nullptr;
    uint16_t* q = dst + i * dst_ld;
    if constexpr (kVec) {
      for (int64_t k = lane * 8; k < dst_ld; k += 256) {
        const uint4 v = p && k < cols ? __ldg(reinterpret_cast<const uint4*>(p + k)) : make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(q + k) = v;
        if constexpr (kMax) {
          larger(v.x), larger(v.y), larger(v.z), larger(v.w);
          larger(v.x >> 16), larger(v.y >> 16), larger(v.z >> 16), larger(v.w >> 16);
        }
      }
    } else {
      for (int64_t k = lane; k < dst_ld; k += 32) {
        const uint16_t v = p && k < cols ? p[k] : (uint16_t)0;
        q[k] = v;
        if constexpr (kMax) larger(v);
      }
    }
  }
  if constexpr (kMax) {
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0 && m) atomicMax(word, m);
  }
}

// ---------------------------------------------------------------------------
// row statistics
// ---------------------------------------------------------------------------

// Rows per block: 8 read whole 32-byte sectors of the partials, and 1024 rows
// still fill the SMs (730 rows of 391 partials: 10 us with 32 rows a block, 7.9 with 8).
constexpr int kStRows = 8;
constexpr int kStSlices = 64;

// (A row with a NaN logit has a NaN maximum, here and below.)
__device__ __forceinline__ void fold(float& m, float& s, float mp, float sp) {
  const float M = fmax_nan(m, mp);
  if (M == -INFINITY) return;
  s = s * exp2f((m - M) * kLog2e) + sp * exp2f((mp - M) * kLog2e);
  m = M;
}

// (max, sum) of the block's kStRows rows over P partials, into sm[0][..], ss[0][..].
__device__ __forceinline__ void fold_rows(const float* __restrict__ part_m, const float* __restrict__ part_s, int64_t P,
                                          int64_t N, int64_t row, bool live, float (*sm)[kStRows],
                                          float (*ss)[kStRows]) {
  float m = -INFINITY, s = 0.f;
  if (live) {
    int64_t p = threadIdx.y;
    for (; p + 3 * kStSlices < P; p += 4 * kStSlices) {  // four loads in flight
      float mp[4], sp[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        mp[u] = part_m[(p + u * kStSlices) * N + row];
        sp[u] = part_s[(p + u * kStSlices) * N + row];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) fold(m, s, mp[u], sp[u]);
    }
    for (; p < P; p += kStSlices) fold(m, s, part_m[p * N + row], part_s[p * N + row]);
  }
  sm[threadIdx.y][threadIdx.x] = m;
  ss[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  for (int h = kStSlices / 2; h >= 1; h >>= 1) {
    if (threadIdx.y < h) {
      float M = sm[threadIdx.y][threadIdx.x], S = ss[threadIdx.y][threadIdx.x];
      fold(M, S, sm[threadIdx.y + h][threadIdx.x], ss[threadIdx.y + h][threadIdx.x]);
      sm[threadIdx.y][threadIdx.x] = M;
      ss[threadIdx.y][threadIdx.x] = S;
    }
    __syncthreads();
  }
}

// logp = (z_t - M) - log S: the target's logit against the row's maximum first,
// so a log-probability near 0 is not the difference of two rounded large numbers.
__global__ void __launch_bounds__(kStRows * kStSlices)
rows_logp_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s, int64_t P, int64_t N,
                 const RowsView R, const float* __restrict__ tgt, float* __restrict__ lse, float* __restrict__ logp) {
  __shared__ float sm[kStSlices][kStRows], ss[kStSlices][kStRows];
  const int64_t row = (int64_t)blockIdx.x * kStRows + threadIdx.x;
  const bool live = row < *R.count;
  fold_rows(part_m, part_s, P, N, row, live, sm, ss);
  if (threadIdx.y == 0 && row < N) {
    const float M = sm[0][threadIdx.x], L = logf(ss[0][threadIdx.x]);
    // (rows behind the count: their softmax is 0)
    lse[row] = live ? M + L : INFINITY;
    if (live) logp[R.row_of[row]] = (tgt[row] - M) - L;
  }
}

// ---------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------

constexpr int kPrepWarps = 4;

// A warp per packed row: the teacher's entries sorted by column, entries of the
// same column joined, absent ones (a column outside of [0, V)) dropped; their
// probabilities; and where each 128-column tile's entries begin.
template <typename TI>
__global__ void __launch_bounds__(kPrepWarps * 32)
topk_prep_kernel(const TI* __restrict__ ids, const float* __restrict__ logp, int K, int K2, int64_t N, int64_t V,
                 float inv_t, int tail, const RowsView R, const TopkView T, float* __restrict__ p_out,
                 float* __restrict__ rest_out) {
  extern __shared__ unsigned long long keys_sh[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long* key = keys_sh + (size_t)warp * K2;
  int32_t* cols = reinterpret_cast<int32_t*>(keys_sh + (size_t)kPrepWarps * K2) + (size_t)warp * K2;
  const int64_t i = (int64_t)blockIdx.x * kPrepWarps + warp;
  const int64_t count = *R.count;
  uint16_t* st = const_cast<uint16_t*>(T.start) + i * T.tiles1;
  if (i >= N) return;
  if (i >= count) {  // no entries
    for (int t = lane; t < T.tiles1; t += 32) st[t] = 0;
    return;
  }
  const int64_t src = (int64_t)R.row_of[i] * K;
  constexpr unsigned long long kNone = 0xffffffffffffffffull;
  float mx = -INFINITY;
  bool nan = false;
  for (int k = lane; k < K2; k += 32) {
    unsigned long long x = kNone;
    if (k < K) {
      const int64_t v = (int64_t)ids[src + k];
      if (v >= 0 && v < V) {
        x = ((unsigned long long)v << 32) | (unsigned)k;
        const float t = logp[src + k];
        mx = fmaxf(mx, t);
        nan = nan || t != t;
      }
    }
    key[k] = x;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  nan = __any_sync(0xffffffffu, nan);
  __syncwarp();
  // bitonic sort by (column, place)
  for (int size = 2; size <= K2; size <<= 1) {
    for (int j = size >> 1; j > 0; j >>= 1) {
      for (int k = lane; k < K2 / 2; k += 32) {
        const int lo = ((k & -j) << 1) | (k & (j - 1)), hi = lo + j;
        const bool up = (lo & size) == 0;
        const unsigned long long x = key[lo], y = key[hi];
        if ((x > y) == up) {
          key[lo] = y;
          key[hi] = x;
        }
      }
      __syncwarp();
    }
  }
  // renormalised: p = e^((t - max) / T) / Z; with a tail: p = e^t
  float z = 0.f;
  if (!tail) {
    for (int k = lane; k < K2; k += 32)
      if (key[k] != kNone) {
        const float t = logp[src + (unsigned)key[k]];
        if (t != -INFINITY) z += expf((t - mx) * inv_t);
      }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (nan) z = NAN;
  }
  int32_t* sid = const_cast<int32_t*>(T.sid) + i * K;
  float* pr = p_out + i * K;
  int n = 0;          // entries of distinct columns so far
  double mass = 0.0;  // this lane's share of the sum of p
  for (int k0 = 0; k0 < K2; k0 += 32) {
    const int k = k0 + lane;
    const unsigned long long x = k < K2 ? key[k] : kNone;
    const bool head = x != kNone && (k == 0 || (key[k - 1] >> 32) != (x >> 32));
    const unsigned heads = __ballot_sync(0xffffffffu, head);
    if (head) {
      double p = 0.0;
      for (int j = k; j < K2 && key[j] != kNone && (key[j] >> 32) == (x >> 32); ++j) {
        const float t = logp[src + (unsigned)key[j]];
        if (tail) p += exp((double)t);
        else if (z != z) p = NAN;
        else if (t != -INFINITY) p += (double)(expf((t - mx) * inv_t) / z);
      }
      const int at = n + __popc(heads & ((1u << lane) - 1u));
      sid[at] = cols[at] = (int32_t)(x >> 32);
      pr[at] = (float)p;
      mass += p;
    }
    n += __popc(heads);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  // what the entries leave over; nothing when every column is listed
  if (lane == 0) {
    const double r = 1.0 - mass;
    rest_out[i] = tail && n > 0 && n < V ? (float)(r > 0.0 ? r : (r == r ? 0.0 : r)) : 0.f;
  }
  __syncwarp();
  for (int t = lane; t < T.tiles1; t += 32) {
    const int64_t col = (int64_t)t * kTopkTile;
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cols[mid] < col) lo = mid + 1;
      else hi = mid;
    }
    st[t] = (uint16_t)lo;
  }
}

// 8 rows per block: the statistics of the columns outside of S are joined, then
// a warp per row takes the K entries: loss, the others' coefficient A, the
// entries' gradients x (in place of their z).
__global__ void __launch_bounds__(kStRows * kStSlices)
distill_rows_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s, int64_t P, int64_t N, int64_t V,
                    const RowsView R, const TopkView T, const float* __restrict__ p_in,
                    const float* __restrict__ rest_in, float* __restrict__ lse_rest, float* __restrict__ A,
                    float* __restrict__ whole_out, float* __restrict__ loss_row, DistillSum* __restrict__ sums) {
  __shared__ float sm[kStSlices][kStRows], ss[kStSlices][kStRows];
  __shared__ double tot[kStRows];
  __shared__ int has[kStRows];
  static_assert(kStRows * 32 <= kStRows * kStSlices, "a warp per row");
  const int64_t row0 = (int64_t)blockIdx.x * kStRows;
  const int64_t count = *R.count;
  fold_rows(part_m, part_s, P, N, row0 + threadIdx.x, row0 + threadIdx.x < count, sm, ss);
  const int tid = threadIdx.y * kStRows + threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int64_t i = row0 + w;
  double loss = 0.0;
  int ok = 0;
  if (w >= kStRows) {
    // (the other warps have joined their slices)
  } else if (i < count) {
    const int n = T.start[i * T.tiles1 + T.tiles1 - 1];
    float* zr = T.z + i * T.K;
    const float* pr = p_in + i * T.K;
    const float rest = rest_in[i];
    const float mr = sm[0][w], sr = ss[0][w];
    float mx = mr, mass = 0.f;
    for (int k = lane; k < n; k += 32) {
      mx = fmax_nan(mx, zr[k]);
      mass += pr[k];
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
    }
    float top = 0.f;
    for (int k = lane; k < n; k += 32) top += exp2f((zr[k] - mx) * kLog2e);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top += __shfl_xor_sync(0xffffffffu, top, o);
    const bool others = n < V && mr != -INFINITY;
    const float sr_mx = others ? sr * exp2f((mr - mx) * kLog2e) : 0.f;
    const float S = top + sr_mx, logS = logf(S);
    // an entry with a column but no mass anywhere (all e^-inf) says nothing
    ok = n > 0 && !(mass == 0.f && rest == 0.f);
    const float whole = mass + rest;
    for (int k = lane; k < n; k += 32) {
      const float p = pr[k], lz = zr[k] - mx;
      if (ok && p != 0.f) loss += (double)(p * (logf(p) - (lz - logS)));
      zr[k] = ok ? whole * (exp2f(lz * kLog2e) / S) - p : 0.f;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
    if (lane == 0) {
      // log q_r from the parts: (mr - mx) + log sr - log S
      if (ok && rest != 0.f)
        loss += others ? (double)(rest * (logf(rest) - ((mr - mx) + logf(sr) - logS))) : (double)INFINITY;
      A[i] = ok && others ? whole * (sr_mx / S) - rest : 0.f;
      lse_rest[i] = others ? mr + logf(sr) : INFINITY;
      whole_out[i] = whole;
      if (loss_row) loss_row[R.row_of[i]] = (float)loss;
    }
  } else if (i < N && lane == 0) {
    A[i] = 0.f;
    lse_rest[i] = INFINITY;
    whole_out[i] = 0.f;
  }
  if (w < kStRows && lane == 0) {
    tot[w] = loss;
    has[w] = ok;
  }
  __syncthreads();
  if (tid == 0) {
    double l = 0.0;
    int n = 0;
#pragma unroll
    for (int r = 0; r < kStRows; ++r) {
      l += tot[r];
      n += has[r];
    }
    sums[blockIdx.x] = DistillSum{l, n};
  }
}

__global__ void __launch_bounds__(256)
distill_final_kernel(const DistillSum* __restrict__ sums, int blocks, int reduction, float* __restrict__ loss,
                     float* __restrict__ weight) {
  __shared__ double l_sh[8], n_sh[8];
  double l = 0.0, n = 0.0;
  for (int b = threadIdx.x; b < blocks; b += 256) {
    l += sums[b].loss;
    n += (double)sums[b].n;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0) {
    l_sh[threadIdx.x >> 5] = l;
    n_sh[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = n = 0.0;
    for (int w = 0; w < 8; ++w) {
      l += l_sh[w];
      n += n_sh[w];
    }
    const double c = reduction == CCE_REDUCE_MEAN ? (n > 0.0 ? n : 1.0) : 1.0;
    if (reduction != CCE_REDUCE_NONE) loss[0] = (float)(l / c);
    weight[0] = (float)(1.0 / c);
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// Bits of |x| as an order of values, 0 for infinities and NaN: a row that holds one
// must not take the scale away from the others.
__device__ __forceinline__ uint32_t finite_bits(uint32_t x) {
  x &= 0x7fffffffu;
  return x < 0x7f800000u ? x : 0u;
}

// The power of two >= m (2^-100 below that) times 2^-14.
__device__ __forceinline__ float scale_of(float m) {
  int ex = -100;
  if (m > 0.f) {
    const float f = frexpf(m, &ex);  // m = f * 2^ex, f in [0.5, 1)
    if (f == 0.5f) --ex;
  }
  return ldexpf(1.f, max(ex, -100) - 14);
}

// One block: per row the power of two above its largest dlogit's bound, |d| (times
// the sum of a teacher's probabilities, where that is above 1), times 2^-14: w / s
// stays below 2^14 in float16, and a softmax value of 2^-28 is still a normal
// number whatever the cotangents of the other rows are.  A row whose bound is not
// finite takes 2^-14 and leaves the largest scale to the others.
__global__ void __launch_bounds__(1024)
rows_scale_kernel(const Cotangent up, const float* __restrict__ whole, const RowsView R, float* __restrict__ rows,
                  float* __restrict__ max_s) {
  __shared__ float red[32];
  const int count = *R.count;
  float m = 0.f;
  for (int i = threadIdx.x; i < (up.per_row || whole ? count : min(count, 1)); i += blockDim.x) {
    const float b = fabsf(up.of(i, R.row_of)) * (whole ? fmaxf(whole[i], 1.f) : 1.f);
    const bool finite = b < INFINITY;
    if (finite) m = fmaxf(m, b);
    if (up.per_row) rows[i] = scale_of(finite ? b : 1.f);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) m = fmaxf(m, red[w]);
    max_s[0] = scale_of(m);
  }
}

// grad_e row n = row pos[n] of each K split's slab added in order, 0 for rows that do not
// count; a warp per row and 128 columns (few rows with many slabs need the width).
template <typename T, bool kVec>
__global__ void __launch_bounds__(256)
rows_scatter_kernel(const float* __restrict__ slabs, const SlabPlan plan, int64_t ld, const RowsView R, int64_t N,
                    int64_t D, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int32_t* pos = R.pos;
  const int64_t tiles = ceil_div(*R.count, 128), stride = tiles * 128 * ld;
  const int num = plan.warp_splits((int)tiles);
  const int64_t pieces = ceil_div(D, 128), items = N * pieces;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < items; i += (int64_t)gridDim.x * 8) {
    const int64_t n = i / pieces, k0 = (i - n * pieces) * 128;
    const int64_t p = pos[n];
    const float* row = slabs + p * ld;
    if constexpr (kVec) {
      const int64_t k = k0 + 4 * lane;
      if (k >= D) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p >= 0) {
        x = *reinterpret_cast<const float4*>(row + k);
#pragma unroll 8
        for (int z = 1; z < num; ++z) {
          const float4 y = *reinterpret_cast<const float4*>(row + z * stride + k);
          x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
      }
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(out + n * D + k) = x;
      } else {
        T h[4] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w)};
        *reinterpret_cast<uint2*>(out + n * D + k) = *reinterpret_cast<uint2*>(h);
      }
    } else {
      for (int64_t k = k0 + lane; k < D && k < k0 + 128; k += 32) {
        float x = 0.f;
        if (p >= 0) {
          x = row[k];
          for (int z = 1; z < num; ++z) x += row[z * stride + k];
        }
        out[n * D + k] = from_f32<T>(x);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// float32 operands as two float16 parts
// ---------------------------------------------------------------------------

// The largest finite |x| as the bits of a float, whatever order the blocks run in.
__global__ void __launch_bounds__(256)
absmax_kernel(const float* __restrict__ x, int64_t rows, int64_t D, const int32_t* __restrict__ row_of,
              const int32_t* __restrict__ count, int vec, uint32_t* __restrict__ word) {
  const int lane = threadIdx.x & 31;
  if (count) rows = min(rows, (int64_t)*count);
  uint32_t m = 0;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const float* p = x + (row_of ? row_of[r] : r) * D;
    if (vec) {
#pragma unroll 8
      for (int64_t k = 4 * lane; k < D; k += 128) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + k));
        m = max(m, max(max(finite_bits(v.x), finite_bits(v.y)), max(finite_bits(v.z), finite_bits(v.w))));
      }
    } else {
      for (int64_t k = lane; k < D; k += 32) m = max(m, finite_bits(__float_as_uint(p[k])));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0 && m) atomicMax(word, m);
}

// s puts the largest value into [2^13, 2^14): hi = fp16(s x), lo = fp16(2^11 (s x - hi)).
// hi has 11 bits down to 2^-14, so of values down to 2^-28 of the largest 22 bits are
// held, and 2^-36 absolute (in units of 1 / s), 2^-50 of the largest, below.  The
// product of two lo's is left out: half as much again there, and 2^-78 of the largest
// values' product where both are that small.  (In hi's own units lo would run out at
// 2^-25, and one row 2^20 above the others would leave them 17 bits.)
// |s x - hi| <= 4, so lo stays below 2^13.
__device__ __forceinline__ void split_parts(float y, __half& hi, __half& lo) {
  hi = __float2half_rn(y);
  lo = __float2half_rn((y - __half2float(hi)) * kLoUnits);
}

__global__ void __launch_bounds__(256)
split_kernel(const float* __restrict__ x, int64_t rows, int64_t D, int64_t Dp, const int32_t* __restrict__ row_of,
             const int32_t* __restrict__ count, int vec, const uint32_t* __restrict__ word, float* __restrict__ scale,
             __half* __restrict__ hi, __half* __restrict__ lo) {
  const int lane = threadIdx.x & 31;
  const float big = __uint_as_float(*word);
  float s = 1.f;
  if (big > 0.f) {
    int ex;
    frexpf(big, &ex);
    s = ldexpf(1.f, min(110, max(-110, 14 - ex)));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    scale[0] = s;
    scale[1] = 1.f / s;
  }
  const int64_t live = count ? min(rows, (int64_t)*count) : rows;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const float* p = r < live ? x + (row_of ? row_of[r] : r) * D : nullptr;
    for (int64_t k = 4 * lane; k < Dp; k += 128) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (p) {
        if (vec && k + 4 <= D) {
          const float4 y = __ldg(reinterpret_cast<const float4*>(p + k));
          v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = k + j < D ? p[k + j] : 0.f;
        }
      }
      __half h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        split_parts(v[j] * s, h[j], l[j]);
      }
      *reinterpret_cast<uint2*>(hi + r * Dp + k) = *reinterpret_cast<uint2*>(h);
      *reinterpret_cast<uint2*>(lo + r * Dp + k) = *reinterpret_cast<uint2*>(l);
    }
  }
}

// grad_c sums s_i (w / s_i) e_i over rows of different scales s_i: e_i takes s_i / S, S the
// largest.  float16: the largest value goes to [2^13, 2^14), so a row 2^20 below the
// largest scale still has normal numbers (e alone would leave 4 bits of them); two
// parts are there already and are split anew.  A warp per row; zeros behind the count.
template <bool kSplit>
__global__ void __launch_bounds__(256)
rows_fold_kernel(const __half* __restrict__ e, const __half* __restrict__ e_lo, int64_t N, int64_t Dk,
                 const int32_t* __restrict__ count, const float* __restrict__ rows, const float* __restrict__ max_s,
                 const uint32_t* __restrict__ word, float* __restrict__ scale, __half* __restrict__ out,
                 __half* __restrict__ out_lo) {
  const int lane = threadIdx.x & 31;
  float k = 1.f;
  if constexpr (!kSplit) {
    const float big = __half2float(__ushort_as_half((unsigned short)*word));
    if (big > 0.f) {
      int ex;
      frexpf(big, &ex);
      k = ldexpf(1.f, 14 - ex);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      scale[0] = k;
      scale[1] = 1.f / k;
    }
  }
  const int64_t live = *count;
  const float inv = 1.f / max_s[0];
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < N; r += (int64_t)gridDim.x * 8) {
    // (at most 1: a row that is not finite may have a scale above the others')
    const float f = r < live ? fminf(rows[r] * inv, 1.f) * k : 0.f;
    for (int64_t c = 4 * lane; c < Dk; c += 128) {
      __half h[4] = {}, l[4] = {};
      if (r < live) {
        *reinterpret_cast<uint2*>(h) = __ldg(reinterpret_cast<const uint2*>(e + r * Dk + c));
        if constexpr (kSplit) *reinterpret_cast<uint2*>(l) = __ldg(reinterpret_cast<const uint2*>(e_lo + r * Dk + c));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kSplit) split_parts((__half2float(h[j]) + __half2float(l[j]) / kLoUnits) * f, h[j], l[j]);
          else h[j] = __float2half_rn(__half2float(h[j]) * f);
        }
      }
      *reinterpret_cast<uint2*>(out + r * Dk + c) = *reinterpret_cast<uint2*>(h);
      if constexpr (kSplit) *reinterpret_cast<uint2*>(out_lo + r * Dk + c) = *reinterpret_cast<uint2*>(l);
    }
  }
}

// grad_bias of a vocabulary chunk from the column sums of 32 rows each, in order:
// the same result every time, where atomics would add in any order.
__global__ void __launch_bounds__(256)
bias_sum_kernel(const float* __restrict__ part, int64_t parts, const int32_t* __restrict__ count, int64_t ld,
                int64_t cols, float* __restrict__ out) {
  __shared__ float sh[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  parts = min(parts, ceil_div(*count, 128) * 4);  // (those of the row tiles that were computed)
  float s = 0.f;
  if (c < cols)
    for (int64_t p = w; p < parts; p += 8) s += part[p * ld + c];
  sh[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][lane];
    out[c] = s;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

unsigned warps_grid(int64_t N) {
  const int64_t b = ceil_div(N, 8);
  return (unsigned)(b < 148 * 8 ? b : 148 * 8);
}

}  // namespace

cudaError_t launch_rows_pack(int64_t N, const void* targets, int target_bytes, int64_t ignore_index, int has_ignore,
                             const uint8_t* mask, const RowsView& R, uint8_t* mask_out, float* per_row_out, float* tgt,
                             uint32_t* words, cudaStream_t s) {
  if (targets == nullptr)
    rows_pack_kernel<void><<<1, kPackThreads, 0, s>>>(nullptr, 0, 0, mask, N, R, mask_out, per_row_out, nullptr,
                                                     words);
  else if (target_bytes == 8)
    rows_pack_kernel<int64_t><<<1, kPackThreads, 0, s>>>((const int64_t*)targets, ignore_index, has_ignore, mask, N, R,
                                                         mask_out, per_row_out, tgt, words);
  else
    rows_pack_kernel<int32_t><<<1, kPackThreads, 0, s>>>((const int32_t*)targets, ignore_index, has_ignore, mask, N, R,
                                                         mask_out, per_row_out, tgt, words);
  return launched();
}

cudaError_t launch_rows_copy(const void* src, int64_t rows, int64_t cols, int64_t src_ld, const RowsView* R, void* dst,
                             int64_t dst_ld, uint32_t* word, cudaStream_t s) {
  const bool vec = ((cols | src_ld | dst_ld) & 7) == 0 && aligned16(src) && aligned16(dst);
  const int32_t* row_of = R ? R->row_of : nullptr;
  const int32_t* count = R ? R->count : nullptr;
  const auto kern = word ? (vec ? rows_copy_kernel<true, true> : rows_copy_kernel<false, true>)
                         : (vec ? rows_copy_kernel<true, false> : rows_copy_kernel<false, false>);
  kern<<<warps_grid(rows), 256, 0, s>>>((const uint16_t*)src, rows, cols, src_ld, row_of, count, (uint16_t*)dst, dst_ld,
                                        word);
  return launched();
}

cudaError_t launch_rows_scale(const Cotangent& up, const float* whole, const RowsView& R, float* rows, float* max_s,
                              cudaStream_t s) {
  rows_scale_kernel<<<1, 1024, 0, s>>>(up, whole, R, rows, max_s);
  return launched();
}

cudaError_t launch_rows_fold(const void* e, const void* e_lo, int64_t N, int64_t Dk, const RowsView& R,
                             const float* rows, const float* max_s, const uint32_t* word, float* scale, void* out,
                             void* out_lo, cudaStream_t s) {
  const __half *h = static_cast<const __half*>(e), *l = static_cast<const __half*>(e_lo);
  if (e_lo) {
    rows_fold_kernel<true><<<warps_grid(N), 256, 0, s>>>(h, l, N, Dk, R.count, rows, max_s, word, scale,
                                                         static_cast<__half*>(out), static_cast<__half*>(out_lo));
    return launched();
  }
  rows_fold_kernel<false><<<warps_grid(N), 256, 0, s>>>(h, nullptr, N, Dk, R.count, rows, max_s, word, scale,
                                                        static_cast<__half*>(out), nullptr);
  return launched();
}

cudaError_t launch_rows_logp(const float* part_m, const float* part_s, int64_t P, int64_t N, const RowsView& R,
                             const float* tgt, float* lse, float* logp, cudaStream_t s) {
  rows_logp_kernel<<<(unsigned)ceil_div(N, kStRows), dim3(kStRows, kStSlices), 0, s>>>(part_m, part_s, P, N, R, tgt, lse,
                                                                                       logp);
  return launched();
}

cudaError_t launch_topk_prep(const void* ids, int id_bytes, const float* logp, int64_t N, int64_t V, int K, double T,
                             int tail, const RowsView& R, const TopkView& topk, float* p, float* rest, cudaStream_t s) {
  int K2 = 2;
  while (K2 < K) K2 *= 2;
  const size_t smem = (size_t)kPrepWarps * K2 * 12;  // at most 48 KB (K <= 1024)
  const unsigned grid = (unsigned)ceil_div(N, kPrepWarps);
  const float inv_t = (float)(1.0 / T);
  if (id_bytes == 8)
    topk_prep_kernel<int64_t><<<grid, kPrepWarps * 32, smem, s>>>((const int64_t*)ids, logp, K, K2, N, V, inv_t, tail, R,
                                                                  topk, p, rest);
  else
    topk_prep_kernel<int32_t><<<grid, kPrepWarps * 32, smem, s>>>((const int32_t*)ids, logp, K, K2, N, V, inv_t, tail, R,
                                                                  topk, p, rest);
  return launched();
}

int64_t distill_blocks(int64_t N) { return ceil_div(N, kStRows); }

cudaError_t launch_distill_rows(const float* part_m, const float* part_s, int64_t P, int64_t N, int64_t V,
                                const RowsView& R, const TopkView& topk, const float* p, const float* rest,
                                int reduction, float* lse_rest, float* A, float* whole, DistillSum* sums, float* loss,
                                float* weight, cudaStream_t s) {
  const int blocks = (int)distill_blocks(N);
  distill_rows_kernel<<<blocks, dim3(kStRows, kStSlices), 0, s>>>(
      part_m, part_s, P, N, V, R, topk, p, rest, lse_rest, A, whole, reduction == CCE_REDUCE_NONE ? loss : nullptr,
      sums);
  cudaError_t err = launched();
  if (err != cudaSuccess) return err;
  distill_final_kernel<<<1, 256, 0, s>>>(sums, blocks, reduction, loss, weight);
  return launched();
}

template <typename T>
static cudaError_t scatter(const float* slabs, const SlabPlan& plan, int64_t ld, const RowsView& R, int64_t N, int64_t D,
                           void* out, cudaStream_t s) {
  const unsigned grid = warps_grid(N * ceil_div(D, 128));
  if (D % 4 == 0 && ld % 4 == 0 && aligned16(slabs) && aligned16(out))
    rows_scatter_kernel<T, true><<<grid, 256, 0, s>>>(slabs, plan, ld, R, N, D, static_cast<T*>(out));
  else
    rows_scatter_kernel<T, false><<<grid, 256, 0, s>>>(slabs, plan, ld, R, N, D, static_cast<T*>(out));
  return launched();
}

cudaError_t launch_rows_scatter(const float* slabs, const SlabPlan& plan, int64_t ld, const RowsView& R, int64_t N,
                                int64_t D, int dtype, void* out, cudaStream_t s) {
  switch (dtype) {
    case CCE_F32: return scatter<float>(slabs, plan, ld, R, N, D, out, s);
    case CCE_F16: return scatter<__half>(slabs, plan, ld, R, N, D, out, s);
    case CCE_BF16: return scatter<__nv_bfloat16>(slabs, plan, ld, R, N, D, out, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_absmax(const float* x, int64_t rows, int64_t D, const RowsView* R, uint32_t* word, cudaStream_t s) {
  if (R == nullptr && rows * D % 4096 == 0) {  // contiguous: rows of a width that keeps many loads in flight
    rows = rows * D / 4096;
    D = 4096;
  }
  absmax_kernel<<<warps_grid(rows), 256, 0, s>>>(x, rows, D, R ? R->row_of : nullptr, R ? R->count : nullptr,
                                                 D % 4 == 0 && aligned16(x), word);
  return launched();
}

cudaError_t launch_split(const float* x, int64_t rows, int64_t D, int64_t Dp, const RowsView* R, const uint32_t* word,
                         float* scale, void* hi, void* lo, cudaStream_t s) {
  split_kernel<<<warps_grid(rows), 256, 0, s>>>(x, rows, D, Dp, R ? R->row_of : nullptr, R ? R->count : nullptr,
                                                D % 4 == 0 && aligned16(x), word, scale, static_cast<__half*>(hi),
                                                static_cast<__half*>(lo));
  return launched();
}

cudaError_t launch_bias_sum(const float* part, int64_t parts, const RowsView& R, int64_t ld, int64_t cols, float* out,
                            cudaStream_t s) {
  bias_sum_kernel<<<(unsigned)ceil_div(cols, 32), 256, 0, s>>>(part, parts, R.count, ld, cols, out);
  return launched();
}

}  // namespace cce
