// The GEMMs of losses on log-probabilities over a batch's packed rows, with
// two-level accumulation.  Part of tc_kernels.cu, after the engine whose
// descriptors, tensor maps and output staging it uses.
//
//   LogitsEpi    z = scale (e c^T + bias): per row and 128-column half the online
//                (max, sum of exp), the target's z, and for the distillation the z
//                of the row's listed columns, which are left out of the sum
//   DlogitsEpi2  the same z for one vocabulary chunk, then the dlogits
//   OutEpi       float32 gradients (float32 inputs)
//
// 320 threads: a TMA warp, an MMA warp and 8 epilogue warps, one CTA per SM over
// a static schedule of (128-row, 256-column) tiles.  There is no filter here: the
// gradients are exact, and rows that do not count are not in the batch.
//
// Why a second level.  tcgen05.mma adds every K = 16 product into its fp32
// accumulator rounding towards zero: a logit of 14 after 144 such steps is
// about 1e-5 too small, always in the same direction, and sums of
// log-probabilities over a sequence add that up.  Here an accumulator holds
// only a segment of K; the epilogue warps add each of those partial logits to
// the total in their registers (128 per thread, round to nearest).  The two TMEM
// accumulators take the segments in turn, so the MMAs run on while the adds are
// made.  A segment of 4 K-blocks (float16 row statistics; segments() has the others)
// is 16 MMAs, about 2000 cycles; its add takes about 500 of the issue slots of the
// 8 epilogue warps.
//
// What is left of the drift is added back in expectation.  A step that rounds
// an accumulator a towards zero loses on average half a unit in its last place,
// 0.72 * 2^-24 |a| (mantissas spread evenly in their logarithm); over the 16
// steps of a partial logit p that grows in a straight line 6 * 2^-24 |p|.  The
// noise on the way makes it less, float16 products (22 bits, cut to the
// accumulator's) make it more.  The partials are multiplied by 1 + k 2^-23 in the
// same fused multiply-add, k (segments() below: a share of the segment's MMA
// steps) from the root mean square error of log-probabilities of 2048 peaked
// rows, V = 32000, in units of 1e-6 for k = 0, 1, 2, 3, 4 at segments of 16 steps
// (float32: 8), in brackets a library's float32 product:
//   bfloat16, D = 2304     1.00 0.68 0.55 0.68 0.98   (5.1)
//   bfloat16, D = 512      1.15 0.80 0.60 0.65 0.92   (2.2)
//   float16, D = 2304      1.31 0.96 0.73 0.64 0.80   (6.5)
//   float16, D = 512       2.30 1.94 1.63 1.37 1.20   (3.1)
//   float32, D = 2304      1.69 1.60 1.63 1.73 1.92   (6.7)
//   float32, D = 512       1.29 1.03 0.93 1.00 1.23   (3.0)
// bfloat16 runs on segments of 32 steps with k = 4: 0.68 (D = 2304), 0.75 (4096),
// 1.08 (512), for half the adds.  With one accumulator for all of K a bfloat16
// D = 2304 head has 5.7.  16-bit gradients and dlogits, which are rounded to 16 bits,
// take segments of 64 steps; float32 products are all summed in segments of 8.
//
// k is a fit to logits that grow steadily.  Where one channel carries a logit alone,
// the cuts that follow it in its segment decide: all of them when it comes first,
// one when it comes last, with the same k 2^-23 added back.  So k lies between the
// two extremes, and what is left is at most 5e-7 of the logit either way: mean errors
// at a logit of 14, first / last in a segment, in units of 1e-6: bfloat16 4.6 / -6.3,
// float16 0.7 / -4.7, float32 -0.3 / -2.8 (one accumulator for D = 4096: 74).
//
// Float32 inputs.  x = (hi + 2^-11 lo) / s with hi, lo float16 and s a power of two that
// puts the tensor's largest value below 2^14: hi holds 11 bits and lo the next 11, of
// values down to 2^-28 of the largest; lo's units are 2^-11 of hi's.
// A product runs as three passes over K, hi hi + hi lo + lo hi (lo lo is 2^-22 of
// it), each on the tensor cores: 3 times the 16-bit work, where FFMA is 20 times
// slower.  512 x 512 x 32000, loss and gradients: 0.37 ms, 2.75 ms on the CUDA cores.
//
// Rows are counted on the device (the batch without its masked rows), so row
// tiles behind the count cost nothing.

constexpr int kRgWarps = 8;                   // epilogue warps: two per TMEM lane quarter, a column half each
constexpr int kRgThreads = 64 + 32 * kRgWarps;
constexpr size_t kRgSmem = 1024 + STAGES * (size_t)STAGE_BYTES + kRgWarps * 4096 + 256;

struct RowsSched {
  const int32_t* rows;   // rows that count, read at the kernel's start
  int64_t N;             // their capacity
  int m_rows, k_rows;    // M / K runs over the rows
  int num_m, num_n, num_kb, ksplit, m_fast, group;
  int b3d = 1;           // MN-major B as one 3-D box (else one 2-D box per 64 columns)
  SlabPlan slabs{};      // cap > 0: K splits by the rows that count
  __device__ __forceinline__ Sched get(int64_t& count) const {
    count = min((int64_t)__ldg(rows), N);
    Sched s{};
    s.num_m = m_rows ? (int)ceil_div(count, BM) : num_m;
    s.num_n = num_n;
    s.num_kb = k_rows ? (int)ceil_div(count, BK) : num_kb;
    s.ksplit = slabs.cap > 0 ? slabs.warp_splits(s.num_m) : ksplit;
    s.m_fast = m_fast;
    s.group = group;
    return s;
  }
};

// What an epilogue thread works on: its row of the tile, and the first of its
// 128 columns.
struct TileAt {
  int64_t row, col0, rows;  // rows: those that count
  int y0, ks, nb;           // first row of the warp's 32, K split, column tile
};

// 2^x, results below the normal range as 0 (they add nothing to a sum that holds a 1)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The bias of a warp's 128 columns: four of them per lane, loaded before the tile's
// products are waited for, and added through the warp's staging area (reads of one
// address by all lanes); with loads beside the adds the logits took 85 instead of
// 80 us, the dlogits 93 instead of 91 (900 rows, D = 1088, V = 50021).
struct Bias128 {
  float b[4];
  template <typename TB>
  __device__ __forceinline__ void load(const void* bias, int64_t col0, int64_t V) {
    if constexpr (!std::is_void<TB>::value) {
      const TB* p = static_cast<const TB*>(bias);
      const int64_t c = col0 + 4 * (threadIdx.x & 31);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = c + j < V ? to_f32(__ldg(p + c + j)) : 0.f;
    }
  }
  // z = us z + bias
  template <typename TB, bool kScaled>
  __device__ __forceinline__ void add(float (&z)[128], float us, const Stager& sg) const {
    if constexpr (!std::is_void<TB>::value) {
      sg.acquire<0>();
      float4* buf = reinterpret_cast<float4*>(sg.buf);
      buf[threadIdx.x & 31] = make_float4(b[0], b[1], b[2], b[3]);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float4 x = buf[j];
        z[4 * j] = (kScaled ? z[4 * j] * us : z[4 * j]) + x.x;
        z[4 * j + 1] = (kScaled ? z[4 * j + 1] * us : z[4 * j + 1]) + x.y;
        z[4 * j + 2] = (kScaled ? z[4 * j + 2] * us : z[4 * j + 2]) + x.z;
        z[4 * j + 3] = (kScaled ? z[4 * j + 3] * us : z[4 * j + 3]) + x.w;
      }
      __syncwarp();
    } else if constexpr (kScaled) {
#pragma unroll
      for (int j = 0; j < 128; ++j) z[j] *= us;
    }
  }
};

// 1 / (s_a s_b) of split operands, 1 for whole ones: s[1] = 1 / s[0]
__device__ __forceinline__ float unscale(const float* a, const float* b) { return a ? a[1] * b[1] : 1.f; }

// The K-blocks that one accumulator holds, of a unit of kb K-blocks walked in
// `passes` passes; no segment spans the first pass, hi hi, and the others, whose
// products are in units of 1 / kLoUnits.
struct Segment {
  int kb, passes, len;
  __device__ __forceinline__ int n() const { return kb * passes; }
  __device__ __forceinline__ int end(int k0) const { return min(k0 < kb ? kb : n(), k0 + len); }
};

struct NoCursor {};

template <typename TB, bool kTopk>
struct LogitsEpi {
  static constexpr int kKind = 0;
  static constexpr bool kStores = false, kExact = true;
  const int32_t* targets;  // [N]
  const void* bias;
  float* part_m;           // [ceil(V / 128)][N]
  float* part_s;
  float* tgt;              // [N]
  int64_t N, V;            // N: the arrays' stride
  float scale;
  const float *se, *sc;    // split operands' scales
  TopkView topk;           // kTopk: the listed columns

  struct State {
    int64_t tl;  // the target's place in this half
    Bias128 bias;
    typename std::conditional<kTopk, TopkCursor, NoCursor>::type cur;
  };
  __device__ __forceinline__ void begin(State& st, const TileAt& t) const {
    const bool live = t.row < t.rows;
    st.bias.template load<TB>(bias, t.col0, V);
    st.tl = -1;
    if constexpr (kTopk) st.cur.open(topk, t.row, live, t.col0 / kTopkTile);
    else if (live) st.tl = (int64_t)targets[t.row] - t.col0;
  }

  __device__ __forceinline__ void finish(State& st, float (&z)[128], const TileAt& t, Stager& sg, const CUtensorMap*) const {
    const bool live = t.row < t.rows;
    const int64_t tl = st.tl;
    // The maximum is kept of the unscaled values; exponents are differences to
    // it first, exact next to the maximum, then one product with scale log2 e.
    float m = -INFINITY, sum = 0.f, tz = 0.f;
    const float cexp = scale * kLog2e;
    if (se) st.bias.template add<TB, true>(z, unscale(se, sc), sg);
    else st.bias.template add<TB, false>(z, 1.f, sg);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t cb = t.col0 + c * 32;
      float* v = z + c * 32;
      if (cb + 32 > V) {
        const int left = (int)(V - cb);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : -INFINITY;
      }
      if constexpr (kTopk) {
        int p;
        const uint32_t bits = st.cur.take(cb, p);
        if (__any_sync(0xffffffffu, bits != 0u)) {
          float* zo = topk.z + t.row * topk.K + p;
#pragma unroll
          for (int g = 0; g < 32; g += 8) {
            if (__any_sync(0xffffffffu, (bits >> g) & 0xffu)) {
#pragma unroll
              for (int j = g; j < g + 8; ++j) {
                if ((bits >> j) & 1u) {
                  zo[__popc(bits & ((1u << j) - 1u))] = v[j] * scale;
                  v[j] = -INFINITY;
                }
              }
            }
          }
        }
      } else {
        const int64_t at = tl - c * 32;
        if (__any_sync(0xffffffffu, at >= 0 && at < 32)) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (at == j) tz = v[j];
        }
      }
      float mc = v[0];
#pragma unroll
      for (int j = 1; j < 32; ++j) mc = fmax_nan(mc, v[j]);
      const float nm = fmax_nan(m, mc);
      if (nm != -INFINITY) {
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) part += ex2((v[j] - nm) * cexp);
        sum = sum * ex2((m - nm) * cexp) + part;
        m = nm;
      }
    }
    if (live) {
      if (t.col0 < V) {
        const int64_t idx = (t.col0 / 128) * N + t.row;
        part_m[idx] = m * scale;
        part_s[idx] = sum;
      }
      if constexpr (!kTopk)
        if (tl >= 0 && tl < 128 && t.col0 + tl < V) tgt[t.row] = tz * scale;
    }
  }
};

// dlogits of one vocabulary chunk (columns relative to it).  Log-probabilities:
// w = d (softmax - onehot).  Distillation: A d e^(z - L) with the coefficient and
// log-sum-exp of the columns outside of the row's list, d x for the listed ones.
// float16 holds w / s, s the row's scale; split: hi + lo.
// 16-bit inputs: w is rounded to their type, as an operand of the gradient products
// must be; half a step beside the result's own half step (bfloat16 gradients are
// 0.0023 to 0.0025 off, 0.0017 with one rounding).  Two parts would double those
// products.
template <typename T, typename TB, bool kTopk, bool kSplit>
struct DlogitsEpi2 {
  static constexpr int kKind = 1;
  static constexpr bool kStores = true, kExact = false;
  const int32_t* targets;
  const float* lse;
  Cotangent up;           // d of a row
  const int32_t* row_of;
  const float* A;         // [N] kTopk: coefficient over d
  const void* bias;       // of column 0 of the whole vocabulary
  RowScale scale;
  float* bias_part;       // [ceil(N / 32)][ld] column sums of w, or nullptr
  int64_t N, V, vc0, vc_end, ld;
  float scale_z;
  const float *se, *sc;
  TopkView topk;

  struct State {
    int64_t tl;      // the target's place in this half
    float G, L, dr;  // dlogits are G e^(z - L); dr: d; both over s
    float s;
    Bias128 bias;
    typename std::conditional<kTopk, TopkCursor, NoCursor>::type cur;
  };
  __device__ __forceinline__ void begin(State& st, const TileAt& t) const {
    const bool live = t.row < t.rows;
    const int64_t v0 = vc0 + t.col0;
    const float d = live ? up.of(t.row, row_of) : 0.f;
    st.bias.template load<TB>(bias, v0, vc_end);
    st.L = live ? lse[t.row] : INFINITY;
    st.s = live ? scale.of(t.row) : 1.f;
    st.dr = d * (1.f / st.s);  // (exact: s is a power of two)
    st.tl = -1;
    if constexpr (kTopk) {
      // (a row that gets no gradient: 0 whatever its coefficient)
      st.G = live && d != 0.f ? A[t.row] * st.dr : 0.f;
      st.cur.open(topk, t.row, live, v0 / kTopkTile);
    } else {
      st.G = st.dr;
      if (live) st.tl = (int64_t)targets[t.row] - v0;
    }
  }

  __device__ __forceinline__ void finish(State& st, float (&z)[128], const TileAt& t, Stager& sg,
                                         const CUtensorMap* tm_lo) const {
    const float G = st.G, L = st.L, dr = st.dr;
    const int64_t v0 = vc0 + t.col0;  // vocabulary id of column 0
    const int64_t tl = st.tl;
    st.bias.template add<TB, kSplit>(z, kSplit ? unscale(se, sc) : 1.f, sg);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t cb = v0 + c * 32;
      float(&v)[32] = *reinterpret_cast<float(*)[32]>(z + c * 32);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = G * ex2((v[j] * scale_z - L) * kLog2e);
      if constexpr (kTopk) {
        int p;
        const uint32_t bits = st.cur.take(cb, p);
        if (__any_sync(0xffffffffu, bits != 0u)) {
          const float* x = topk.z + t.row * topk.K + p;
#pragma unroll
          for (int g = 0; g < 32; g += 8) {
            if (__any_sync(0xffffffffu, (bits >> g) & 0xffu)) {
#pragma unroll
              for (int j = g; j < g + 8; ++j)
                if ((bits >> j) & 1u) v[j] = dr * __ldg(x + __popc(bits & ((1u << j) - 1u)));
            }
          }
        }
      } else {
        const int64_t at = tl - c * 32;
        if (__any_sync(0xffffffffu, at >= 0 && at < 32)) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (at == j) v[j] -= G;
        }
      }
      if (cb + 32 > vc_end) {  // (products of stored columns with rows of c behind the chunk)
        const int left = (int)(vc_end - cb);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : 0.f;
      }
      if (t.y0 < N && cb < vc_end) {
        if (bias_part != nullptr) {
          float x[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = v[j] * st.s;
          const int lane = threadIdx.x & 31;
          const float colsum = warp_transpose_sum32(x);
          if (cb + lane < vc_end) bias_part[(int64_t)(t.y0 / 32) * ld + (cb - vc0) + lane] = colsum;
        }
        sg.template store16<T>(v, (int)(cb - vc0), t.y0);
        if constexpr (kSplit) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = (v[j] - to_f32(from_f32<T>(v[j]))) * kLoUnits;
          const CUtensorMap* tm_hi = sg.tm;
          sg.tm = tm_lo;
          sg.template store16<T>(v, (int)(cb - vc0), t.y0);
          sg.tm = tm_hi;
        }
      }
    }
  }
};

// out[row][col] = f1 f2 (A B) in T
template <typename T>
struct Out16Epi {
  static constexpr int kKind = 3;
  static constexpr bool kStores = true, kExact = false;
  const float *f1, *f2;
  int64_t M, D;

  struct State {};
  __device__ __forceinline__ void begin(State&, const TileAt&) const {}
  __device__ __forceinline__ void finish(State&, float (&z)[128], const TileAt& t, Stager& sg, const CUtensorMap*) const {
    const float s = (f1 ? *f1 : 1.f) * (f2 ? *f2 : 1.f);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t col = t.col0 + c * 32;
      if (col >= D || t.y0 >= M) continue;
      float(&v)[32] = *reinterpret_cast<float(*)[32]>(z + c * 32);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= s;
      sg.template store16<T>(v, (int)col, t.y0);
    }
  }
};

// out[row][col] (+)= f1 f2 (A B), float32, f1 by row; K split ks behind ks times the row tiles
struct OutEpi {
  static constexpr bool kStores = true, kExact = false;
  RowScale f1;
  const float* f2;
  int add;
  int64_t M, D;
  int kind;  // slot in g_mma_cols
  static constexpr int kKind = -1;  // (that of `kind`)

  struct State {};
  __device__ __forceinline__ void begin(State&, const TileAt&) const {}
  __device__ __forceinline__ void finish(State&, float (&z)[128], const TileAt& t, Stager& sg, const CUtensorMap*) const {
    const float f = (t.row < t.rows || !f1.per_row ? f1.of(t.row) : 1.f) * (f2 ? *f2 : 1.f);
    const int y = t.ks * (int)round_up(t.rows, BM) + t.y0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t col = t.col0 + c * 32;
      if (col >= D || t.y0 >= M) continue;
      float(&v)[32] = *reinterpret_cast<float(*)[32]>(z + c * 32);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= f;
      sg.store_f32(v, (int)col, y, 0, add != 0);
    }
  }
};

template <bool A_MN, bool B_MN, bool kSplit, class Epi>
__global__ void __launch_bounds__(kRgThreads, 1)
rows_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA2,
                 const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmB2,
                 const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmC2, const RowsSched rs,
                 const Epi epi, const uint32_t idesc, const int seg_kb, const float untruncate) {
  constexpr int kPasses = kSplit ? 3 : 1;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* sA = smem_raw + pad;
  uint8_t* sB = sA + STAGES * A_BYTES;
  uint8_t* sOut = sB + STAGES * B_BYTES;  // 4 KB per epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + kRgWarps * 4096);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int64_t rows;
  const Sched sched = rs.get(rows);
  const int units = sched.units();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + i, 1);
      mbar_init(tempty + i, 32 * kRgWarps);
    }
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        int mb, nb, ks, kb0, kb1;
        sched.coords(u, mb, nb, ks);
        sched.krange(ks, kb0, kb1);
        for (int p = 0; ok && p < kPasses; ++p) {  // hi hi, hi lo, lo hi
          const CUtensorMap* ma = p == 2 ? &tmA2 : &tmA;
          const CUtensorMap* mb_ = p == 1 ? &tmB2 : &tmB;
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(empty + stage, phase ^ 1u, 11)) { ok = false; break; }
            uint8_t* a = sA + stage * A_BYTES;
            uint8_t* b = sB + stage * B_BYTES;
            mbar_arrive_expect_tx(full + stage, STAGE_BYTES);
            if constexpr (A_MN) tma_load_3d(a, ma, full + stage, 0, kb * BK, mb * (BM / 64));
            else tma_load_2d(a, ma, full + stage, kb * BK, mb * BM);
            if constexpr (B_MN) {
              if (rs.b3d) {
                tma_load_3d(b, mb_, full + stage, 0, kb * BK, nb * (BN / 64));
              } else {
#pragma unroll
                for (int j = 0; j < BN / 64; ++j)
                  tma_load_2d(b + j * BOX_MN_BYTES, mb_, full + stage, nb * BN + j * 64, kb * BK);
              }
            } else tma_load_2d(b, mb_, full + stage, kb * BK, nb * BN);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      unsigned long long mma_cols = 0;
      const uint64_t adesc0 = A_MN ? smem_desc(smem_u32(sA), BOX_MN_BYTES, 1024) : smem_desc(smem_u32(sA), 16, 1024);
      const uint64_t bdesc0 = B_MN ? smem_desc(smem_u32(sB), BOX_MN_BYTES, 1024) : smem_desc(smem_u32(sB), 16, 1024);
      constexpr uint32_t a_kstep = (A_MN ? 2048u : 32u) >> 4;
      constexpr uint32_t b_kstep = (B_MN ? 2048u : 32u) >> 4;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        int mb, nb, ks, kb0, kb1;
        sched.coords(u, mb, nb, ks);
        sched.krange(ks, kb0, kb1);
        const Segment seg{kb1 - kb0, kPasses, seg_kb};
        for (int k0 = 0, k1; ok && k0 < seg.n(); k0 = k1) {
          k1 = seg.end(k0);
          if (!mbar_wait(tempty + acc, acc_phase ^ 1u, 12)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + (uint32_t)(acc * BN);
          uint32_t fresh = 1;
          for (int k = k0; k < k1; ++k) {
            if (!mbar_wait(full + stage, phase, 13)) { ok = false; break; }
            tc_fence_after();
            const uint64_t ad = adesc0 + (uint64_t)((stage * A_BYTES) >> 4);
            const uint64_t bd = bdesc0 + (uint64_t)((stage * B_BYTES) >> 4);
#pragma unroll
            for (int i = 0; i < BK / 16; ++i) {
              mma_f16(d, ad + i * a_kstep, bd + i * b_kstep, idesc, fresh ^ 1u);
              fresh = 0;
            }
            mma_cols += (BK / 16) * BN;
            mma_commit(empty + stage);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          mma_commit(tfull + acc);
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
      if constexpr (Epi::kKind >= 0) atomicAdd(&g_mma_cols[Epi::kKind], mma_cols);
      else atomicAdd(&g_mma_cols[epi.kind], mma_cols);
    }
    __syncwarp();
  } else {
    // ---------------- epilogue ----------------
    const int q = warp & 3;           // TMEM lane quarter of this warp
    const int h = (warp - 2) >> 2;    // column half
    const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * 128);
    Stager sg{&tmC, sOut + (warp - 2) * 4096, 0};
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
      int mb, nb, ks, kb0, kb1;
      sched.coords(u, mb, nb, ks);
      sched.krange(ks, kb0, kb1);
      const Segment seg{kb1 - kb0, kPasses, seg_kb};
      const int y0 = mb * BM + q * 32;
      const TileAt t{(int64_t)y0 + lane, (int64_t)nb * BN + h * 128, rows, y0, ks, nb};
      typename Epi::State st;
      epi.begin(st, t);
      float z[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) z[j] = 0.f;
#pragma unroll 1
      for (int k0 = 0; k0 < seg.n(); k0 = seg.end(k0)) {
        // (one verdict for the warp: the TMEM reads below need all of its lanes)
        ok = __all_sync(0xffffffffu, mbar_wait(tfull + acc, acc_phase, 14));
        if (!ok) break;
        tc_fence_after();
        const float f = kSplit && k0 >= seg.kb ? untruncate / kLoUnits : untruncate;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tmem_ld32(tbase + (uint32_t)(acc * BN + c * 32), v);
#pragma unroll
          for (int j = 0; j < 32; ++j) z[c * 32 + j] = fmaf(v[j], f, z[c * 32 + j]);
        }
        tc_fence_before();
        mbar_arrive(tempty + acc);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) break;
      epi.finish(st, z, t, sg, &tmC2);
    }
    if constexpr (Epi::kStores) sg.drain();  // output boxes written before the kernel ends
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---- host side ----

struct RowsMaps {
  CUtensorMap A, A2, B, B2, C, C2;
};

// K-blocks (64 columns) per accumulator segment, and what its partial products are
// multiplied by (see the top of this file).  `exact`: row statistics.
struct Segments {
  int kb;
  float untruncate;
};

Segments segments(bool exact, bool split, bool bf16, int64_t num_kb) {
  const int kb = split ? 2 : !exact ? 16 : bf16 ? 8 : 4;
  const float steps = 4.f * (float)(num_kb < kb ? num_kb : kb);
  const float units = roundf(steps * (split ? 1.f / 4 : bf16 ? 1.f / 8 : 3.f / 16));
  return Segments{kb, 1.f + units * 1.1920929e-7f};
}

template <bool A_MN, bool B_MN, bool kSplit, class Epi>
cudaError_t rows_gemm(const RowsMaps& m, const RowsSched& rs, const Epi& epi, bool bf16, int64_t max_units,
                      cudaStream_t s) {
  auto kern = rows_gemm_kernel<A_MN, B_MN, kSplit, Epi>;
  static std::atomic<unsigned long long> attr_ctx[64];
  cudaError_t err = ensure_smem_attr(kern, kRgSmem, attr_ctx);
  if (err != cudaSuccess) return err;
  if (max_units <= 0) return cudaSuccess;
  const int grid = max_units < num_sms() ? (int)max_units : num_sms();
  const Segments sg = segments(Epi::kExact, kSplit, bf16, rs.k_rows ? ceil_div(rs.N, BK) : rs.num_kb);
  kern<<<grid, kRgThreads, kRgSmem, s>>>(m.A, m.A2, m.B, m.B2, m.C, m.C2, rs, epi, instr_desc(BM, BN, bf16, A_MN, B_MN),
                                         sg.kb, sg.untruncate);
  return launched();
}

// e (packed rows) and the chunk's rows of c, K-major: whole 16-bit operands or hi / lo.
bool ec_maps(RowsMaps& m, const RowsGemmArgs& a) {
  const bool bf16 = a.dtype == CCE_BF16, split = a.dtype == CCE_F32;
  const int64_t off = a.vc0 * a.Dk;
  bool ok = make_tmap(&m.A, a.e, bf16, a.Dk, a.N, a.Dk, BK, BM) &&
            make_tmap(&m.B, static_cast<const uint16_t*>(a.c) + off, bf16, a.Dk, a.vc_len, a.Dk, BK, BN);
  m.A2 = m.A;
  m.B2 = m.B;
  if (split)
    ok = ok && make_tmap(&m.A2, a.e_lo, bf16, a.Dk, a.N, a.Dk, BK, BM) &&
         make_tmap(&m.B2, static_cast<const uint16_t*>(a.c_lo) + off, bf16, a.Dk, a.vc_len, a.Dk, BK, BN);
  m.C = m.C2 = m.A;  // (replaced where an epilogue stores)
  return ok;
}

// Schedule of the two logits kernels: row tiles first, so that a column tile of c
// is read once for all of them.
RowsSched ec_sched(const RowsGemmArgs& a) {
  return RowsSched{a.R.count, a.N, 1, 0, 0, (int)ceil_div(a.vc_len, BN), (int)ceil_div(a.Dk, BK), 1, 1,
                   raster_group(a.N * a.Dk * 2)};
}

template <typename TB, bool kTopk>
cudaError_t logits_launch(const RowsGemmArgs& a, cudaStream_t s) {
  RowsMaps m;
  if (!ec_maps(m, a)) return cudaErrorInvalidValue;
  const RowsSched rs = ec_sched(a);
  const LogitsEpi<TB, kTopk> epi{a.R.targets, a.bias, a.part_m, a.part_s, a.tgt, a.N, a.V, a.scale_z, a.se, a.sc, a.topk};
  const int64_t units = ceil_div(a.N, BM) * rs.num_n;
  return a.dtype == CCE_F32 ? rows_gemm<false, false, true>(m, rs, epi, false, units, s)
                            : rows_gemm<false, false, false>(m, rs, epi, a.dtype == CCE_BF16, units, s);
}

template <typename TB>
cudaError_t logits_dispatch(const RowsGemmArgs& a, cudaStream_t s) {
  return a.topk.sid ? logits_launch<TB, true>(a, s) : logits_launch<TB, false>(a, s);
}

template <typename T, typename TB, bool kTopk, bool kSplit>
cudaError_t dlogits2_launch(const RowsGemmArgs& a, cudaStream_t s) {
  RowsMaps m;
  const int dt = a.dtype == CCE_BF16 ? CCE_BF16 : CCE_F16;
  if (!ec_maps(m, a) || !make_tmap_out(&m.C, a.dl, dt, a.vc_len, a.N, a.vc_ld)) return cudaErrorInvalidValue;
  m.C2 = m.C;
  if (kSplit && !make_tmap_out(&m.C2, a.dl_lo, dt, a.vc_len, a.N, a.vc_ld)) return cudaErrorInvalidValue;
  const RowsSched rs = ec_sched(a);
  const DlogitsEpi2<T, TB, kTopk, kSplit> epi{a.R.targets, a.lse, a.up, a.R.row_of, a.A, a.bias, a.scale, a.bias_part,
                                             a.N, a.V, a.vc0, a.vc0 + a.vc_len, a.vc_ld, a.scale_z, a.se, a.sc, a.topk};
  return rows_gemm<false, false, kSplit>(m, rs, epi, dt == CCE_BF16, ceil_div(a.N, BM) * rs.num_n, s);
}

template <typename TB, bool kTopk>
cudaError_t dlogits2_types(const RowsGemmArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case CCE_F32: return dlogits2_launch<__half, TB, kTopk, true>(a, s);
    case CCE_F16: return dlogits2_launch<__half, TB, kTopk, false>(a, s);
    case CCE_BF16: return dlogits2_launch<__nv_bfloat16, TB, kTopk, false>(a, s);
  }
  return cudaErrorNotSupported;
}

template <typename TB>
cudaError_t dlogits2_dispatch(const RowsGemmArgs& a, cudaStream_t s) {
  return a.topk.sid ? dlogits2_types<TB, true>(a, s) : dlogits2_types<TB, false>(a, s);
}

// float32 [rows][ld] output of D columns, written in (16 x 32 x 1) boxes
bool make_tmap_f32(CUtensorMap* tm, const float* out, int64_t D, int64_t ld, int64_t rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)rows, 1};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * 4), (cuuint64_t)(rows * ld * 4)};
  cuuint32_t box[3] = {16, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(out), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kSplit>
cudaError_t grad_e_rows(const RowsGemmArgs& a, float* slabs, const SlabPlan& plan, bool accumulate, cudaStream_t s) {
  const bool bf16 = a.dtype == CCE_BF16;
  const int64_t off = a.vc0 * a.Dk;
  RowsMaps m;
  int b3d = 0;
  bool ok = make_tmap(&m.A, a.dl, bf16, a.vc_len, a.N, a.vc_ld, BK, BM) &&
            make_tmap_mn(&m.B, static_cast<const uint16_t*>(a.c) + off, bf16, a.Dk, a.vc_len, a.Dk, BN / 64, &b3d) &&
            make_tmap_f32(&m.C, slabs, a.Dout, a.Dout, (int64_t)plan.cap * BM);
  m.A2 = m.A, m.B2 = m.B, m.C2 = m.C;
  if (kSplit)
    ok = ok && make_tmap(&m.A2, a.dl_lo, bf16, a.vc_len, a.N, a.vc_ld, BK, BM) &&
         make_tmap_mn(&m.B2, static_cast<const uint16_t*>(a.c_lo) + off, bf16, a.Dk, a.vc_len, a.Dk, BN / 64, &b3d);
  if (!ok) return cudaErrorInvalidValue;
  const RowsSched rs{a.R.count, a.N, 1, 0, 0, plan.num_n, (int)ceil_div(a.vc_len, BK), 1, 1,
                     raster_group(a.N * a.vc_len * 2), b3d, plan};
  const OutEpi epi{a.scale, kSplit ? a.sc + 1 : nullptr, accumulate ? 1 : 0, a.N, a.Dout, 2};
  return rows_gemm<false, true, kSplit>(m, rs, epi, bf16, (int64_t)plan.cap * plan.num_n, s);
}

// grad_c rows of the chunk.  T: the output's type (float with split operands)
template <typename T, bool kSplit>
cudaError_t grad_c_rows(const RowsGemmArgs& a, void* grad_c, cudaStream_t s) {
  const bool bf16 = a.dtype == CCE_BF16;
  T* out = static_cast<T*>(grad_c) + a.vc0 * a.Dout;
  const int64_t cols = round_up(a.vc_len, 64);  // (rows of grad_c behind the chunk are clipped by the output's map)
  RowsMaps m;
  int b3d = 0;
  const void *e = a.ec ? a.ec : a.e, *e_lo = a.ec ? a.ec_lo : a.e_lo;
  bool ok = make_tmap_mn3d(&m.A, a.dl, bf16, cols, a.N, a.vc_ld, BK, BM / 64) &&
            make_tmap_mn(&m.B, e, bf16, a.Dk, a.N, a.Dk, BN / 64, &b3d);
  m.A2 = m.A, m.B2 = m.B;
  if constexpr (kSplit)
    ok = ok && make_tmap_mn3d(&m.A2, a.dl_lo, bf16, cols, a.N, a.vc_ld, BK, BM / 64) &&
         make_tmap_mn(&m.B2, e_lo, bf16, a.Dk, a.N, a.Dk, BN / 64, &b3d) &&
         make_tmap_f32(&m.C, out, a.Dout, a.Dout, a.vc_len);
  else
    ok = ok && make_tmap_out(&m.C, out, a.dtype, a.Dout, a.vc_len, a.Dout);
  if (!ok) return cudaErrorInvalidValue;
  m.C2 = m.C;
  const int num_m = (int)ceil_div(a.vc_len, BM), num_n = (int)ceil_div(a.Dout, BN);
  const RowsSched rs{a.R.count, a.N, 0, 1, num_m, num_n, 0, 1, 0, raster_group(a.N * a.Dk * 2), b3d};
  if constexpr (kSplit) {
    const OutEpi epi{RowScale{a.max_s, 0}, a.se + 1, 0, a.vc_len, a.Dout, 3};
    return rows_gemm<true, true, true>(m, rs, epi, bf16, (int64_t)num_m * num_n, s);
  } else {
    const Out16Epi<T> epi{a.max_s, a.sec ? a.sec + 1 : nullptr, a.vc_len, a.Dout};
    return rows_gemm<true, true, false>(m, rs, epi, bf16, (int64_t)num_m * num_n, s);
  }
}
