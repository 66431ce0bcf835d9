// Losses on per-token log-probabilities: the clipped policy loss with a KL
// term, and the preference loss of (chosen, rejected) sequence pairs.
//
// Tokens lie in one array of N; sequence s holds the tokens [cu[s], cu[s+1])
// (packed) or [s L, (s+1) L) (padded rows).  Tokens that the mask or the
// offsets leave out add nothing and get a zero gradient, whatever they hold
// (infinities, NaN): values are taken or left, never multiplied by the mask.
//
// Policy loss of a token with d = logp - old, r = e^d, advantage A:
//     l = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (e^q - 1 - q),  q = ref - logp
//     dl/dlogp = -r A (where the minimum is not the clipped side) - beta (e^q - 1)
// Which side is taken is decided on d against log(1 - lo) and log(1 + hi), in 64
// bits next to them: r rounded to 32 bits would give some token of a large batch
// the other side's gradient.
//
// Preference loss of a pair with D_s = sum over tokens of (logp - ref):
//     gap = D_chosen - D_rejected, h = beta gap - margin;
//     sigmoid -(1-ls) log s(h) - ls log s(-h), hinge max(0, 1 - h), ipo (gap - 1/(2 beta))^2
//     dloss/dlogp_t = +- slope (1 / length when normalised), the same for every token of a sequence.
//
// The least is to read the inputs once (17 bytes per token for a float32 policy
// loss with a KL term); up to a million tokens launches and the host take longer.
// 8.4 million tokens, float32, advantages per token: forward 50 us (3.2 TB/s, 74%
// of the issue slots: two exponentials, the series and the borders are some 100
// instructions a token), join 5.5, backward 11.  6.3 million bfloat16 tokens in
// 1024 pairs: 33, 9 and 16 us.
// One pass reads the tokens in chunks of 1024 or 4096; per-sequence sums are joined
// from the chunks' pieces in a fixed order by a second launch (the same launch
// when there is one chunk), so results do not depend on scheduling.  Sums are
// held in 64 bits from the first join on.
#include "kernels.cuh"

namespace cce {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;                    // consecutive tokens of a thread: one 16-byte load of float32
constexpr int kStep = kThreads * kPer;     // tokens of a block at a time
// A block takes one step, or kMany of a large batch: finding its sequences and
// adding its sums up (microseconds of latency) then cost a quarter of a token's
// share; 64 k tokens in 16 blocks would leave most SMs idle.
constexpr int kMany = 4;
constexpr int64_t kManyFrom = 2ll * 148 * 8 * kStep;  // tokens: two waves of 8 blocks an SM
constexpr int kCached = 64;                // sequence offsets of a block's tokens kept in shared memory
constexpr int kWarps = kThreads / 32;
constexpr int kGroup = 8;                  // lanes that join the pieces of one sequence
constexpr int kFinalSeqs = kThreads / kGroup;  // sequences (pairs) a block of the second launch takes at a time
constexpr int kFinalBlocks = 148;

// Offsets of the sequences, clamped into the array so that no offset read from
// memory ever becomes an address outside of it.
struct Seqs {
  const int32_t* cu;  // [S + 1], nullptr: rows of `len` tokens
  int64_t S, len, N;
  int64_t chunk;      // tokens of a block
  __device__ __forceinline__ int64_t bound(int64_t s) const {
    if (cu == nullptr) return s * len;
    const int64_t b = __ldg(cu + s);
    return b < 0 ? 0 : (b > N ? N : b);
  }
  // First sequence in [lo, hi] that ends behind token t (hi if none before it does).
  __device__ __forceinline__ int64_t find(int64_t lo, int64_t hi, int64_t t) const {
    if (cu == nullptr) return len > 0 ? (t / len < S ? t / len : S) : S;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (bound(mid + 1) <= t) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  }
  // find(0, S, t) by a whole warp, 32 offsets a step: 3 dependent loads for
  // 32,768 sequences where one thread's search needs 15.
  __device__ __forceinline__ int64_t find_warp(int64_t t) const {
    if (cu == nullptr) return find(0, S, t);
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, hi = S;
    while (hi > lo) {
      const int64_t n = hi - lo;
      const int64_t step = (n + 31) / 32;
      const int64_t p = lo + (lane + 1) * step - 1;  // the lane's pivot
      const bool before = p < hi && bound(p + 1) <= t;
      const int64_t cnt = __popc(__ballot_sync(0xffffffffu, before));
      const int64_t base = lo;
      lo = base + cnt * step < hi ? base + cnt * step : hi;
      hi = base + (cnt + 1) * step - 1 < hi ? base + (cnt + 1) * step - 1 : hi;
      if (hi < lo) hi = lo;
    }
    return lo;
  }
};

// The pieces of per-sequence sums: a sequence's piece in the chunk where it
// begins, and every chunk's piece of the sequence that began before it.
struct Pieces {
  double* begin;    // [S]
  double* head;     // [chunks]
  int32_t* begin_n; // tokens counted
  int32_t* head_n;
};

struct BlockSums {  // a chunk's totals
  double loss, kl;
  int32_t n, clipped;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, int i, int n, bool vec, float (&v)[kPer]) {
  if (vec && i + kPer <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p + i));
      const T* h = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = to_f32(h[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = i + j < n ? to_f32(p[i + j]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, int i, int n, bool vec, const float (&v)[kPer]) {
  if (vec && i + kPer <= n) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint2 x;
      T* h = reinterpret_cast<T*>(&x);
#pragma unroll
      for (int j = 0; j < kPer; ++j) h[j] = from_f32<T>(v[j]);
      *reinterpret_cast<uint2*>(p + i) = x;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i + j < n) p[i + j] = from_f32<T>(v[j]);
  }
}

__device__ __forceinline__ void load_mask4(const uint8_t* m, int i, int n, bool vec, bool (&on)[kPer]) {
  if (m == nullptr) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) on[j] = i + j < n;
  } else if (vec && i + kPer <= n) {
    const uchar4 x = __ldg(reinterpret_cast<const uchar4*>(m + i));
    on[0] = x.x != 0, on[1] = x.y != 0, on[2] = x.z != 0, on[3] = x.w != 0;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) on[j] = i + j < n && m[i + j] != 0;
  }
}

template <typename X>
__device__ __forceinline__ X warp_sum(X v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sequences lo .. hi that a block's tokens [c0, c1) lie in, and (unless they
// are many: most blocks hold a piece of one or two) where each begins in them.
struct ChunkSeqs {
  int64_t lo, hi;
  int cut[kCached];  // begin of sequence lo + k, from c0, clamped to [0, c1 - c0]
  __device__ __forceinline__ bool cached() const { return hi - lo + 2 <= kCached; }
  // All threads of the block; ends with a barrier.
  __device__ __forceinline__ void load(const Seqs& q, int64_t c0, int64_t c1) {
    const int warp = threadIdx.x >> 5;
    if (warp < 2) {
      const int64_t s = q.find_warp(warp == 0 ? c0 : c1 - 1);
      if ((threadIdx.x & 31) == 0) (warp == 0 ? lo : hi) = s;
    }
    __syncthreads();
    if (hi < lo) {  // (offsets that decrease)
      __syncthreads();
      if (threadIdx.x == 0) hi = lo;
      __syncthreads();
    }
    if (cached()) {
      if (threadIdx.x <= hi - lo + 1) {
        const int64_t b = lo + threadIdx.x <= q.S ? q.bound(lo + threadIdx.x) : c0;
        cut[threadIdx.x] = (int)(b < c0 ? 0 : b > c1 ? c1 - c0 : b - c0);
      }
      __syncthreads();
    }
  }
};

// Sequences of the thread's tokens t .. t + 3 of the block (-1: none); true when
// all four lie in one, s[0].
__device__ __forceinline__ bool token_seqs(const Seqs& q, const ChunkSeqs& cs, int64_t c0, int t, int64_t (&s)[kPer]) {
  if (cs.cached()) {
    const int n = (int)(cs.hi - cs.lo);
    int k = 0, end = n;
    while (k < end) {  // first sequence that ends behind token t
      const int mid = (k + end) >> 1;
      if (cs.cut[mid + 1] <= t) k = mid + 1;
      else end = mid;
    }
    const bool some = cs.lo + k < q.S;
    if (some && cs.cut[k] <= t && t + kPer <= cs.cut[k + 1]) {
      s[0] = cs.lo + k;
      return true;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      while (k < n && cs.cut[k + 1] <= t + j) ++k;
      s[j] = cs.lo + k < q.S && cs.cut[k] <= t + j && t + j < cs.cut[k + 1] ? cs.lo + k : -1;
    }
    return false;
  }
  int64_t cur = q.find(cs.lo, cs.hi, c0 + t);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    while (cur < cs.hi && q.bound(cur + 1) <= c0 + t + j) ++cur;
    s[j] = cur < q.S && q.bound(cur) <= c0 + t + j && c0 + t + j < q.bound(cur + 1) ? cur : -1;
  }
  return false;
}

// Sums of val (0 and off for tokens that do not count) over the pieces that
// the block's sequences have in its tokens: a warp per sequence, or where they
// are few several warps a sequence, each a part of the piece.  All threads of
// the block; `sh` holds kWarps of each.
__device__ __forceinline__ void piece_sums(const Seqs& q, const ChunkSeqs& cs, int64_t c0, int64_t c1, const float* val,
                                           const uint8_t* on, double* shd, int* shi, const Pieces& out) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t hi = cs.hi < q.S ? cs.hi : q.S - 1;
  const int64_t num = hi - cs.lo + 1;
  const int parts = num <= 1 ? kWarps : num <= 2 ? kWarps / 2 : num <= 4 ? kWarps / 4 : 1;
  const int part = warp % parts;
  for (int64_t s0 = cs.lo; s0 <= hi; s0 += kWarps / parts) {
    const int64_t s = s0 + warp / parts;
    double v = 0.0;
    int n = 0;
    bool some = false, begins = false;
    if (s <= hi) {
      const int64_t a = q.bound(s), b = q.bound(s + 1);
      const int t0 = (int)((a > c0 ? a : c0) - c0), t1 = (int)((b < c1 ? b : c1) - c0);
      some = t1 > t0;
      begins = a >= c0;
      // a lane's values in float32 by 4, then in 64 bits
      for (int t = t0 + part * 32 + lane; t < t1; t += 4 * 32 * parts) {
        float x = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (t + 32 * parts * u < t1) {
            x += val[t + 32 * parts * u];
            n += on[t + 32 * parts * u];
          }
        }
        v += (double)x;
      }
      v = warp_sum(v);
      n = warp_sum(n);
    }
    if (parts > 1) {
      __syncthreads();
      if (lane == 0) {
        shd[warp] = v;
        shi[warp] = n;
      }
      __syncthreads();
      if (lane == 0 && part == 0) {
        for (int k = 1; k < parts; ++k) {
          v += shd[warp + k];
          n += shi[warp + k];
        }
      }
    }
    if (lane == 0 && part == 0 && some) {
      if (begins) {
        out.begin[s] = v;
        out.begin_n[s] = n;
      } else {
        out.head[c0 / q.chunk] = v;
        out.head_n[c0 / q.chunk] = n;
      }
    }
  }
}

// Sum and count of sequence s from its pieces, by kGroup lanes (all get them).
__device__ __forceinline__ void join(const Seqs& q, const Pieces& p, int64_t s, double& v, int& n) {
  v = 0.0;
  n = 0;
  const int g = threadIdx.x & (kGroup - 1);
  const int64_t a = s < q.S ? q.bound(s) : 0, b = s < q.S ? q.bound(s + 1) : 0;
  if (b > a) {
    const int64_t b0 = a / q.chunk, b1 = (b - 1) / q.chunk;
    if (g == 0) {
      v = p.begin[s];
      n = p.begin_n[s];
    }
    for (int64_t k = b0 + 1 + g; k <= b1; k += kGroup) {
      v += p.head[k];
      n += p.head_n[k];
    }
  }
#pragma unroll
  for (int o = kGroup / 2; o >= 1; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
}

// Sum over the block's threads, in a fixed order; thread 0 has it.
template <typename X>
__device__ __forceinline__ X block_sum(X v, X* sh) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  X r = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < kWarps; ++w) r += sh[w];
  return r;
}

// Whether this is the last of the grid's blocks to get here (all threads of
// it; the others' writes are visible then).  `counter` was zeroed by an
// earlier launch.
__device__ __forceinline__ bool last_block(unsigned* counter, int* sh) {
  if (gridDim.x == 1) {
    __syncthreads();
    return true;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *sh = atomicAdd(counter, 1u) == gridDim.x - 1;
  __syncthreads();
  __threadfence();
  return *sh != 0;
}

// ---------------------------------------------------------------------------
// policy loss
// ---------------------------------------------------------------------------

struct Policy {
  const void* logp;
  const void* old;   // nullptr: the policy itself (ratio 1)
  const void* ref;   // nullptr: no KL term
  const float* adv;
  const uint8_t* mask;
  Seqs q;
  int adv_token;     // advantages per token, else per sequence
  int reduction;     // CCE_REDUCE_*
  int vec;
  float lo, hi, dual, beta;        // clipped ratios, dual clip (0: none), KL weight
  double log_lo, log_hi, log_dual;
  // outputs
  float* loss;       // [1], per token for CCE_REDUCE_NONE
  float* stats;      // [2] mean KL, share of clipped tokens
  float* coef;       // [N] dl/dlogp before the reduction's weights
  float* weight;     // [1] weight of a token, [1 + S] and of its sequence
  // workspace
  BlockSums* blk;
  Pieces pc;
  double* part;      // [kFinalBlocks][2]
  unsigned* counter;
  int chunks;
};

struct TokenOut {
  float loss, g, kl;
  bool clipped;
};

// e^q - 1 - q and e^q - 1.  Below |q| = 1 the first from its series to q^11 (the
// next term is 4e-9 of it): the difference would cancel.  Both are computed and
// one is taken: in a warp of tokens some are always far from the reference.
__device__ __forceinline__ void kl3(float q, float& kl, float& em1) {
  float p = 1.f / 39916800.f;
  p = fmaf(p, q, 1.f / 3628800.f);
  p = fmaf(p, q, 1.f / 362880.f);
  p = fmaf(p, q, 1.f / 40320.f);
  p = fmaf(p, q, 1.f / 5040.f);
  p = fmaf(p, q, 1.f / 720.f);
  p = fmaf(p, q, 1.f / 120.f);
  p = fmaf(p, q, 1.f / 24.f);
  p = fmaf(p, q, 1.f / 6.f);
  p = fmaf(p, q, 0.5f);
  const float near = q * q * p, far = expf(q) - 1.f;
  const bool small = fabsf(q) < 1.f;
  kl = small ? near : far - q;
  em1 = small ? q + near : far;
}

// Whether d = x - old lies above (below) the border, decided on the exact difference:
// d is rounded to float32, so only next to the border are 64 bits needed.
__device__ __forceinline__ bool beyond(bool above, float d, float x, float old, double border) {
  const float b = (float)border;
  if (fabsf(d - b) <= 1e-6f * (1.f + fabsf(d))) {
    const double e = (double)x - (double)old;
    return above ? e > border : e < border;
  }
  return above ? d > b : d < b;
}

__device__ __forceinline__ TokenOut policy_token(const Policy& P, float x, float old, float ref, float A) {
  // (without old the ratio is 1; a NaN log-probability stays one)
  const float d = P.old ? x - old : (x == x ? 0.f : x);
  if (!P.old) old = x;
  // (an advantage of 0 asks nothing of a ratio past float32's range, e^88.7: its
  // product is 0 whatever finite number stands here, and NaN stays)
  const float r = A == 0.f ? d : expf(d);
  const bool pos = A > 0.f, neg = A < 0.f;
  TokenOut o;
  // the advantage's sign says which border can be passed
  o.clipped = (pos || neg) && beyond(pos, d, x, old, pos ? P.log_hi : P.log_lo);
  float bounded = o.clipped ? (pos ? P.hi : P.lo) : r;
  if (P.dual > 0.f) {
    const bool far = neg && beyond(true, d, x, old, P.log_dual);
    bounded = far ? P.dual : bounded;
    o.clipped = o.clipped || far;
  }
  o.loss = -(bounded * A);
  o.g = o.clipped ? 0.f : -(r * A);
  o.kl = 0.f;
  if (P.ref) {
    float em1;
    kl3(ref - x, o.kl, em1);
    if (P.beta != 0.f) {  // (0: the term is only measured, and may pass float32's range)
      o.loss = fmaf(P.beta, o.kl, o.loss);
      o.g = fmaf(-P.beta, em1, o.g);
    }
  }
  return o;
}

// The second half of the forward pass: per-sequence sums to the loss and the weights.
__device__ void policy_final(const Policy& P) {
  __shared__ double shd[kWarps];
  __shared__ int shi[kWarps];
  __shared__ int last;
  double total = 0.0;
  int seqs = 0;
  if (P.reduction == CCE_REDUCE_SEQUENCE) {
    for (int64_t s0 = (int64_t)blockIdx.x * kFinalSeqs; s0 < P.q.S; s0 += (int64_t)gridDim.x * kFinalSeqs) {
      const int64_t s = s0 + threadIdx.x / kGroup;
      double v;
      int n;
      join(P.q, P.pc, s, v, n);
      if (s < P.q.S && (threadIdx.x & (kGroup - 1)) == 0) {
        P.weight[1 + s] = n > 0 ? 1.f / (float)n : 0.f;
        if (n > 0) {
          total += v / n;
          ++seqs;
        }
      }
    }
    total = block_sum(total, shd);
    seqs = block_sum(seqs, shi);
    if (gridDim.x > 1) {
      if (threadIdx.x == 0) {
        P.part[2 * blockIdx.x] = total;
        P.part[2 * blockIdx.x + 1] = (double)seqs;
      }
      if (!last_block(P.counter, &last)) return;
      if (threadIdx.x == 0) {
        total = 0.0;
        seqs = 0;
        for (unsigned b = 0; b < gridDim.x; ++b) {
          total += P.part[2 * b];
          seqs += (int)P.part[2 * b + 1];
        }
      }
    }
  }
  // totals over the chunks (the last or only block)
  double loss = 0.0, kl = 0.0, n = 0.0, clipped = 0.0;
#pragma unroll 4
  for (int b = threadIdx.x; b < P.chunks; b += kThreads) {
    const BlockSums x = P.blk[b];
    loss += x.loss;
    kl += x.kl;
    n += (double)x.n;
    clipped += (double)x.clipped;
  }
  loss = block_sum(loss, shd);
  kl = block_sum(kl, shd);
  n = block_sum(n, shd);
  clipped = block_sum(clipped, shd);
  if (threadIdx.x == 0) {
    const double cnt = n > 0.0 ? n : 1.0;
    P.stats[0] = (float)(kl / cnt);
    P.stats[1] = (float)(clipped / cnt);
    if (P.reduction == CCE_REDUCE_MEAN) {
      P.loss[0] = (float)(loss / cnt);
      P.weight[0] = (float)(1.0 / cnt);
    } else if (P.reduction == CCE_REDUCE_SUM) {
      P.loss[0] = (float)loss;
      P.weight[0] = 1.f;
    } else if (P.reduction == CCE_REDUCE_SEQUENCE) {
      const double m = seqs > 0 ? (double)seqs : 1.0;
      P.loss[0] = (float)(total / m);
      P.weight[0] = (float)(1.0 / m);
    } else {
      P.weight[0] = 1.f;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) policy_forward_kernel(const Policy P) {
  __shared__ __align__(16) float val[kMany * kStep];
  __shared__ __align__(4) uint8_t on_sh[kMany * kStep];
  __shared__ ChunkSeqs cs;
  __shared__ double shd[kWarps];
  __shared__ int shi[kWarps];
  const int64_t N = P.q.N;
  const int64_t c0 = (int64_t)blockIdx.x * P.q.chunk;
  const int64_t c1 = c0 + P.q.chunk < N ? c0 + P.q.chunk : N;
  const bool by_seq = P.reduction == CCE_REDUCE_SEQUENCE;
  const bool search = by_seq || !P.adv_token;
  const bool vec = P.vec != 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *P.counter = 0u;
  int64_t b0 = 0, b1 = N;  // tokens before the first and behind the last sequence
  if (search) {
    cs.load(P.q, c0, c1);
  } else if (P.q.cu != nullptr) {
    b0 = P.q.S > 0 ? P.q.bound(0) : N;
    b1 = P.q.S > 0 ? P.q.bound(P.q.S) : N;
  }
  float loss = 0.f, kl = 0.f;  // of the thread's few tokens
  int n = 0, clipped = 0;
  const int len = (int)(c1 - c0);
  const T* logp = static_cast<const T*>(P.logp) + c0;
  const T* oldp = static_cast<const T*>(P.old) + c0;
  const T* refp = static_cast<const T*>(P.ref) + c0;
#pragma unroll 1
  for (int i = threadIdx.x * kPer; i < len; i += kStep) {
    float x[kPer], old[kPer] = {}, ref[kPer] = {}, A[kPer] = {};
    bool on[kPer];
    load4(logp, i, len, vec, x);
    load_mask4(P.mask ? P.mask + c0 : nullptr, i, len, vec, on);
    if (P.old) load4(oldp, i, len, vec, old);
    if (P.ref) load4(refp, i, len, vec, ref);
    if (P.adv_token) load4(P.adv + c0, i, len, vec, A);
    if (search) {
      int64_t s[kPer];
      if (token_seqs(P.q, cs, c0, i, s)) {
        if (!P.adv_token) A[0] = A[1] = A[2] = A[3] = __ldg(P.adv + s[0]);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          on[j] = on[j] && s[j] >= 0;
          if (!P.adv_token) A[j] = on[j] ? __ldg(P.adv + s[j]) : 0.f;
        }
      }
    } else if (P.q.cu != nullptr) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) on[j] = on[j] && c0 + i + j >= b0 && c0 + i + j < b1;
    }
    float l[kPer], g[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      // (computed for every token, taken where it counts: what a masked one holds goes nowhere)
      const TokenOut o = policy_token(P, x[j], old[j], ref[j], A[j]);
      l[j] = on[j] ? o.loss : 0.f;
      g[j] = on[j] ? o.g : 0.f;
      loss += l[j];
      kl += on[j] ? o.kl : 0.f;
      n += on[j];
      clipped += on[j] && o.clipped;
    }
    store4(P.coef + c0, i, len, vec, g);
    if (P.reduction == CCE_REDUCE_NONE) store4(P.loss + c0, i, len, vec, l);
    if (by_seq) {
      *reinterpret_cast<float4*>(val + i) = make_float4(l[0], l[1], l[2], l[3]);
      *reinterpret_cast<uchar4*>(on_sh + i) = make_uchar4(on[0], on[1], on[2], on[3]);
    }
  }
  if (by_seq) {
    __syncthreads();
    piece_sums(P.q, cs, c0, c1, val, on_sh, shd, shi, P.pc);
  }
  const double loss_sum = block_sum((double)loss, shd), kl_sum = block_sum((double)kl, shd);
  n = block_sum(n | clipped << 16, shi);  // (at most 4096 tokens a block)
  if (threadIdx.x == 0) P.blk[blockIdx.x] = BlockSums{loss_sum, kl_sum, n & 0xffff, n >> 16};
  if (gridDim.x == 1) {
    __syncthreads();
    policy_final(P);
  }
}

__global__ void __launch_bounds__(kThreads) policy_final_kernel(const Policy P) { policy_final(P); }

// grad = upstream * weight * coef: 4 bytes read and one value written per token.
template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_backward_kernel(const float* __restrict__ coef, const float* __restrict__ weight, const float* __restrict__ up,
                       int up_token, int by_seq, const Seqs q, int vec, T* __restrict__ grad) {
  __shared__ ChunkSeqs cs;
  const int64_t c0 = (int64_t)blockIdx.x * q.chunk;
  const int64_t c1 = c0 + q.chunk < q.N ? c0 + q.chunk : q.N;
  const float w = (up_token ? 1.f : __ldg(up)) * __ldg(weight);
  if (by_seq) cs.load(q, c0, c1);
  const int len = (int)(c1 - c0);
#pragma unroll 1
  for (int i = threadIdx.x * kPer; i < len; i += kStep) {
    float g[kPer], u[kPer];
    load4(coef + c0, i, len, vec != 0, g);
    if (up_token) load4(up + c0, i, len, vec != 0, u);
    if (by_seq) {
      int64_t s[kPer];
      if (token_seqs(q, cs, c0, i, s)) {
        const float ws = __ldg(weight + 1 + s[0]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) g[j] = g[j] != 0.f ? g[j] * ws : 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) g[j] = s[j] >= 0 && g[j] != 0.f ? g[j] * __ldg(weight + 1 + s[j]) : 0.f;
      }
    }
    // (a token that does not count has coef 0: an infinite upstream must not make it NaN)
#pragma unroll
    for (int j = 0; j < kPer; ++j) g[j] = g[j] == 0.f ? 0.f : g[j] * w * (up_token ? u[j] : 1.f);
    store4(grad + c0, i, len, vec != 0, g);
  }
}

// ---------------------------------------------------------------------------
// preference loss
// ---------------------------------------------------------------------------

struct Preference {
  const void* logp;
  const void* ref;        // per token, logp's type; nullptr: none
  const float* ref_seq;   // per sequence (a sum over its tokens); nullptr: none
  const uint8_t* mask;
  Seqs q;                 // S = 2 pairs: sequence p is chosen, pairs + p rejected
  int64_t pairs;
  int kind, reduction, by_length, vec;
  double beta, margin, smoothing;
  float* loss;            // [1], [pairs] for CCE_REDUCE_NONE
  float* rewards;         // [2 pairs] beta D
  float* coef;            // [2 pairs] dloss/dlogp of a token of the sequence
  Pieces pc;
  double* part;
  unsigned* counter;
};

// The pairs' losses and slopes from the sequences' sums.
__device__ void preference_final(const Preference& P) {
  __shared__ double shd[kWarps];
  __shared__ int last;
  double total = 0.0;
  for (int64_t p0 = (int64_t)blockIdx.x * kFinalSeqs; p0 < P.pairs; p0 += (int64_t)gridDim.x * kFinalSeqs) {
    const int64_t p = p0 + threadIdx.x / kGroup;
    double dw = 0.0, dl = 0.0;
    int nw = 0, nl = 0;
    join(P.q, P.pc, p < P.pairs ? p : P.q.S, dw, nw);
    join(P.q, P.pc, p < P.pairs ? P.pairs + p : P.q.S, dl, nl);
    if (p < P.pairs && (threadIdx.x & (kGroup - 1)) == 0) {
      if (P.ref_seq) {
        dw -= (double)P.ref_seq[p];
        dl -= (double)P.ref_seq[P.pairs + p];
      }
      const double iw = P.by_length ? 1.0 / (nw > 0 ? nw : 1) : 1.0;
      const double il = P.by_length ? 1.0 / (nl > 0 ? nl : 1) : 1.0;
      dw *= iw;
      dl *= il;
      const double gap = dw - dl, beta = P.beta, h = beta * gap - P.margin;
      double loss, slope;  // slope = dloss/dgap
      if (P.kind == CCE_PREF_SIGMOID) {
        // log s(h) = -(max(-h, 0) + log1p(e^-|h|)); 64 bits: a few per pair
        const double t = log1p(exp(-fabs(h)));
        const double ls = P.smoothing;
        loss = (1.0 - ls) * (fmax(-h, 0.0) + t) + ls * (fmax(h, 0.0) + t);
        slope = beta * (ls - 1.0 / (1.0 + exp(h)));
      } else if (P.kind == CCE_PREF_HINGE) {
        loss = h < 1.0 ? 1.0 - h : (h >= 1.0 ? 0.0 : h);  // (NaN stays NaN)
        slope = h < 1.0 ? -beta : 0.0;
      } else {
        const double d = gap - 0.5 / beta;
        loss = d * d;
        slope = 2.0 * d;
      }
      total += loss;
      if (P.reduction == CCE_REDUCE_NONE) P.loss[p] = (float)loss;
      if (P.reduction == CCE_REDUCE_MEAN) slope /= (double)P.pairs;
      P.coef[p] = (float)(slope * iw);
      P.coef[P.pairs + p] = (float)(-slope * il);
      P.rewards[p] = (float)(beta * dw);
      P.rewards[P.pairs + p] = (float)(beta * dl);
    }
  }
  total = block_sum(total, shd);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) P.part[blockIdx.x] = total;
    if (!last_block(P.counter, &last)) return;
    if (threadIdx.x == 0) {
      total = 0.0;
      for (unsigned b = 0; b < gridDim.x; ++b) total += P.part[b];
    }
  }
  if (threadIdx.x == 0 && P.reduction != CCE_REDUCE_NONE)
    P.loss[0] = (float)(P.reduction == CCE_REDUCE_MEAN ? total / (double)P.pairs : total);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) preference_forward_kernel(const Preference P) {
  __shared__ __align__(16) float val[kMany * kStep];
  __shared__ __align__(4) uint8_t on_sh[kMany * kStep];
  __shared__ ChunkSeqs cs;
  __shared__ double shd[kWarps];
  __shared__ int shi[kWarps];
  const int64_t N = P.q.N;
  const int64_t c0 = (int64_t)blockIdx.x * P.q.chunk;
  const int64_t c1 = c0 + P.q.chunk < N ? c0 + P.q.chunk : N;
  const bool vec = P.vec != 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *P.counter = 0u;
  const int len = (int)(c1 - c0);
  const T* logp = static_cast<const T*>(P.logp) + c0;
  const T* refp = static_cast<const T*>(P.ref) + c0;
#pragma unroll 2
  for (int i = threadIdx.x * kPer; i < len; i += kStep) {
    float x[kPer], ref[kPer];
    bool on[kPer];
    load4(logp, i, len, vec, x);
    load_mask4(P.mask ? P.mask + c0 : nullptr, i, len, vec, on);
    if (P.ref) load4(refp, i, len, vec, ref);
    float d[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) d[j] = on[j] ? (P.ref ? x[j] - ref[j] : x[j]) : 0.f;
    *reinterpret_cast<float4*>(val + i) = make_float4(d[0], d[1], d[2], d[3]);
    *reinterpret_cast<uchar4*>(on_sh + i) = make_uchar4(on[0], on[1], on[2], on[3]);
  }
  cs.load(P.q, c0, c1);  // (ends with a barrier: val and on_sh are complete)
  piece_sums(P.q, cs, c0, c1, val, on_sh, shd, shi, P.pc);
  if (gridDim.x == 1) {
    __syncthreads();
    preference_final(P);
  }
}

__global__ void __launch_bounds__(kThreads) preference_final_kernel(const Preference P) { preference_final(P); }

template <typename T>
__global__ void __launch_bounds__(kThreads)
preference_backward_kernel(const float* __restrict__ coef, const float* __restrict__ up, int up_pair, int64_t pairs,
                           const uint8_t* __restrict__ mask, const Seqs q, int vec, T* __restrict__ grad) {
  __shared__ ChunkSeqs cs;
  const int64_t c0 = (int64_t)blockIdx.x * q.chunk;
  const int64_t c1 = c0 + q.chunk < q.N ? c0 + q.chunk : q.N;
  cs.load(q, c0, c1);
  const int len = (int)(c1 - c0);
  auto slope = [&](int64_t s) { return __ldg(coef + s) * __ldg(up + (up_pair ? (s < pairs ? s : s - pairs) : 0)); };
#pragma unroll 1
  for (int i = threadIdx.x * kPer; i < len; i += kStep) {
    bool on[kPer];
    load_mask4(mask ? mask + c0 : nullptr, i, len, vec != 0, on);
    int64_t s[kPer];
    float g[kPer];
    if (token_seqs(q, cs, c0, i, s)) {
      const float x = slope(s[0]);
#pragma unroll
      for (int j = 0; j < kPer; ++j) g[j] = on[j] ? x : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) g[j] = on[j] && s[j] >= 0 ? slope(s[j]) : 0.f;
    }
    store4(grad + c0, i, len, vec != 0, g);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Workspace shared by both losses: block totals, pieces, the second launch's
// partials and its counter.
struct Carve {
  BlockSums* blk;
  Pieces pc;
  double* part;
  unsigned* counter;
};

Carve carve(void* ws, int64_t S, int64_t chunks) {
  char* p = static_cast<char*>(ws);
  Carve c;
  auto take = [&](size_t bytes) {
    char* r = p;
    p += up256(bytes);
    return r;
  };
  c.blk = reinterpret_cast<BlockSums*>(take(chunks * sizeof(BlockSums)));
  c.pc.begin = reinterpret_cast<double*>(take(S * sizeof(double)));
  c.pc.head = reinterpret_cast<double*>(take(chunks * sizeof(double)));
  c.pc.begin_n = reinterpret_cast<int32_t*>(take(S * sizeof(int32_t)));
  c.pc.head_n = reinterpret_cast<int32_t*>(take(chunks * sizeof(int32_t)));
  c.part = reinterpret_cast<double*>(take(2 * kFinalBlocks * sizeof(double)));
  c.counter = reinterpret_cast<unsigned*>(take(sizeof(unsigned)));
  return c;
}

int final_blocks(int64_t items) {
  const int64_t b = ceil_div(items > 0 ? items : 1, kFinalSeqs);
  return (int)(b < kFinalBlocks ? b : kFinalBlocks);
}

}  // namespace

static int64_t chunk_of(int64_t N) { return N >= kManyFrom ? kMany * kStep : kStep; }
// (an empty batch still has a chunk: it zeroes the second launch's counter)
static int64_t chunks_of(int64_t N) { return N > 0 ? ceil_div(N, chunk_of(N)) : 1; }

// Runs launch(type tag) for a dtype.
template <typename F>
static cudaError_t by_type(int dtype, F launch) {
  switch (dtype) {
    case CCE_F32: launch(float()); break;
    case CCE_F16: launch(__half()); break;
    case CCE_BF16: launch(__nv_bfloat16()); break;
    default: return cudaErrorInvalidValue;
  }
  return launched();
}

size_t token_loss_workspace_bytes(int64_t N, int64_t S) {
  const int64_t chunks = chunks_of(N);
  return up256(chunks * sizeof(BlockSums)) + up256(S * 8) + up256(chunks * 8) + up256(S * 4) + up256(chunks * 4) +
         up256(2 * kFinalBlocks * 8) + up256(sizeof(unsigned));
}

cudaError_t policy_forward(const PolicyArgs& a, void* ws, cudaStream_t s) {
  Policy P{};
  P.logp = a.logp, P.old = a.old, P.ref = a.ref, P.adv = a.adv, P.mask = a.mask;
  P.q = Seqs{a.cu, a.S, a.S > 0 ? a.N / a.S : 0, a.N, chunk_of(a.N)};
  P.adv_token = a.adv_token, P.reduction = a.reduction;
  P.lo = (float)(1.0 - a.clip_low), P.hi = (float)(1.0 + a.clip_high), P.dual = (float)a.dual_clip;
  P.beta = (float)a.kl_coef;
  P.log_lo = log1p(-a.clip_low), P.log_hi = log1p(a.clip_high), P.log_dual = a.dual_clip > 0 ? log(a.dual_clip) : 0.0;
  P.loss = a.loss, P.stats = a.stats, P.coef = a.coef, P.weight = a.weight;
  P.chunks = (int)chunks_of(a.N);
  const Carve c = carve(ws, a.S, P.chunks);
  P.blk = c.blk, P.pc = c.pc, P.part = c.part, P.counter = c.counter;
  P.vec = aligned16(a.logp) && aligned16(a.old) && aligned16(a.ref) && aligned16(a.mask) && aligned16(a.coef) &&
          (!a.adv_token || aligned16(a.adv)) && (a.reduction != CCE_REDUCE_NONE || aligned16(a.loss));
  cudaError_t err = by_type(a.dtype, [&](auto t) {
    policy_forward_kernel<decltype(t)><<<P.chunks, kThreads, 0, s>>>(P);
  });
  if (err != cudaSuccess || P.chunks == 1) return err;
  policy_final_kernel<<<a.reduction == CCE_REDUCE_SEQUENCE ? final_blocks(a.S) : 1, kThreads, 0, s>>>(P);
  return launched();
}

cudaError_t policy_backward(const float* coef, const float* weight, const float* up, int up_token, int reduction,
                            const int32_t* cu, int64_t N, int64_t S, int dtype, void* grad, cudaStream_t s) {
  const Seqs q{cu, S, S > 0 ? N / S : 0, N, chunk_of(N)};
  const int by_seq = reduction == CCE_REDUCE_SEQUENCE;
  const int vec = aligned16(coef) && aligned16(grad) && (!up_token || aligned16(up));
  return by_type(dtype, [&](auto t) {
    policy_backward_kernel<decltype(t)><<<(int)chunks_of(N), kThreads, 0, s>>>(
        coef, weight, up, up_token, by_seq, q, vec, static_cast<decltype(t)*>(grad));
  });
}

cudaError_t preference_forward(const PreferenceArgs& a, void* ws, cudaStream_t s) {
  Preference P{};
  const int64_t S = 2 * a.pairs;
  P.logp = a.logp, P.ref = a.ref, P.ref_seq = a.ref_seq, P.mask = a.mask;
  P.q = Seqs{a.cu, S, S > 0 ? a.N / S : 0, a.N, chunk_of(a.N)};
  P.pairs = a.pairs, P.kind = a.kind, P.reduction = a.reduction, P.by_length = a.by_length;
  P.beta = a.beta, P.margin = a.margin, P.smoothing = a.smoothing;
  P.loss = a.loss, P.rewards = a.rewards, P.coef = a.coef;
  const int chunks = (int)chunks_of(a.N);
  const Carve c = carve(ws, S, chunks);
  P.pc = c.pc, P.part = c.part, P.counter = c.counter;
  P.vec = aligned16(a.logp) && aligned16(a.ref) && aligned16(a.mask);
  cudaError_t err = by_type(a.dtype, [&](auto t) {
    preference_forward_kernel<decltype(t)><<<chunks, kThreads, 0, s>>>(P);
  });
  if (err != cudaSuccess || chunks == 1) return err;
  preference_final_kernel<<<final_blocks(a.pairs), kThreads, 0, s>>>(P);
  return launched();
}

cudaError_t preference_backward(const float* coef, const float* up, int up_pair, const uint8_t* mask, const int32_t* cu,
                                int64_t N, int64_t pairs, int dtype, void* grad, cudaStream_t s) {
  const Seqs q{cu, 2 * pairs, pairs > 0 ? N / (2 * pairs) : 0, N, chunk_of(N)};
  const int vec = aligned16(mask) && aligned16(grad);
  return by_type(dtype, [&](auto t) {
    preference_backward_kernel<decltype(t)><<<(int)chunks_of(N), kThreads, 0, s>>>(
        coef, up, up_pair, pairs, mask, q, vec, static_cast<decltype(t)*>(grad));
  });
}

}  // namespace cce
