// Row statistics of the logits with two-level accumulation (16-bit inputs), for
// the losses that need log-probabilities to float32 accuracy.  Part of
// tc_kernels.cu, after the engine whose descriptors and tensor maps it uses.
//
// Per (128-row, 256-column) tile: z = scale (e c^T + bias), and per row over each
// 128-column half the online (max, sum of exp), the target's z, and for the
// distillation the z of the row's listed columns, which are left out of the sum.
//
// Why a second level.  tcgen05.mma adds every K = 16 product into its fp32
// accumulator rounding towards zero: a logit of 14 after 144 such steps is
// about 1e-5 too small, always in the same direction, and sums of
// log-probabilities over a sequence add that up.  Here an accumulator holds
// only kSegKb K-blocks (256 products); the epilogue warps add each of those
// partial logits to the total in their registers (128 per thread, round to
// nearest).  The two TMEM accumulators take the segments in turn, so the MMAs
// never wait for the adds: a segment's 16 MMAs take about 2000 cycles, its add
// about 500 of the issue slots of the 8 epilogue warps.
//
// What is left of the drift is added back in expectation.  A step that rounds
// an accumulator a towards zero loses on average half a unit in its last place,
// 0.72 * 2^-24 |a| (mantissas spread evenly in their logarithm); over the 16
// steps of a partial logit p that grows in a straight line 6 * 2^-24 |p|.  The
// noise on the way makes it less: the drift measured on two heads is 3.1 and
// 3.6 * 2^-24 |p|.  kUntruncate multiplies the partials by 1 + 4 * 2^-24, in the
// same fused multiply-add.  Errors of the log-probabilities of a D = 2304 head
// (mean; root mean square), 1434 rows: one accumulator -4.7e-6 (5.7e-6),
// segments -1.1e-6 (1.5e-6), and corrected 1e-7 (0.9e-6); a library's float32
// product 9e-9 (5.0e-6).
//
// Rows are counted on the device (the batch without its masked rows), so row
// tiles behind the count cost nothing.

template <typename TB>
struct LogitsArgs {
  const int32_t* rows;     // rows that count, read at the kernel's start
  const int32_t* targets;  // [N]
  const void* bias;
  float* part_m;           // [ceil(V / 128)][N]
  float* part_s;
  float* tgt;              // [N]
  int64_t N, V;            // N: the arrays' stride
  int num_n, num_kb, group;
  float scale;
  TopkView topk;           // kTopk: the listed columns
};

constexpr int kLgWarps = 8;                   // epilogue warps: two per TMEM lane quarter, a column half each
constexpr int kLgThreads = 64 + 32 * kLgWarps;
constexpr int kSegKb = 4;                              // K-blocks per accumulator segment
constexpr float kUntruncate = 1.f + 2.f * 1.1920929e-7f;  // for kSegKb = 4
constexpr size_t kLgSmem = 1024 + STAGES * (size_t)STAGE_BYTES + 256;

// 2^x, results below the normal range as 0 (they add nothing to a sum that holds a 1)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename TB, bool kTopk>
__global__ void __launch_bounds__(kLgThreads, 1)
tc_logits_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const LogitsArgs<TB> a, const uint32_t idesc) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* sA = smem_raw + pad;
  uint8_t* sB = sA + STAGES * A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + STAGES * B_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t rows = min((int64_t)__ldg(a.rows), a.N);
  Sched sched{};
  sched.num_m = (int)ceil_div(rows, BM);
  sched.num_n = a.num_n;
  sched.m_fast = 1;
  sched.group = a.group;
  const int num_tiles = sched.num_m * a.num_n;
  const int segs = (a.num_kb + kSegKb - 1) / kSegKb;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + i, 1);
      mbar_init(tempty + i, 32 * kLgWarps);
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
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
        int mb, nb, ks;
        sched.coords(t, mb, nb, ks);
        for (int kb = 0; kb < a.num_kb; ++kb) {
          if (!mbar_wait(empty + stage, phase ^ 1u, 11)) { ok = false; break; }
          mbar_arrive_expect_tx(full + stage, STAGE_BYTES);
          tma_load_2d(sA + stage * A_BYTES, &tmA, full + stage, kb * BK, mb * BM);
          tma_load_2d(sB + stage * B_BYTES, &tmB, full + stage, kb * BK, nb * BN);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      unsigned long long mma_cols = 0;
      const uint64_t adesc0 = smem_desc(smem_u32(sA), 16, 1024);
      const uint64_t bdesc0 = smem_desc(smem_u32(sB), 16, 1024);
      bool ok = true;
      for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
        for (int s = 0; ok && s < segs; ++s) {
          if (!mbar_wait(tempty + acc, acc_phase ^ 1u, 12)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + (uint32_t)(acc * BN);
          const int kb1 = min(a.num_kb, (s + 1) * kSegKb);
          uint32_t fresh = 1;
          for (int kb = s * kSegKb; kb < kb1; ++kb) {
            if (!mbar_wait(full + stage, phase, 13)) { ok = false; break; }
            tc_fence_after();
            const uint64_t ad = adesc0 + (uint64_t)((stage * A_BYTES) >> 4);
            const uint64_t bd = bdesc0 + (uint64_t)((stage * B_BYTES) >> 4);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              mma_f16(d, ad + k * 2, bd + k * 2, idesc, fresh ^ 1u);
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
      atomicAdd(&g_mma_cols[0], mma_cols);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;           // TMEM lane quarter of this warp
    const int h = (warp - 2) >> 2;    // column half
    const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * 128);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
      int mb, nb, ks;
      sched.coords(t, mb, nb, ks);
      const int64_t row = (int64_t)mb * BM + q * 32 + lane;
      const bool live = row < rows;
      const int64_t col0 = (int64_t)nb * BN + h * 128;
      float z[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) z[j] = 0.f;
#pragma unroll 1
      for (int s = 0; s < segs; ++s) {
        // (one verdict for the warp: the TMEM reads below need all of its lanes)
        ok = __all_sync(0xffffffffu, mbar_wait(tfull + acc, acc_phase, 14));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tmem_ld32(tbase + (uint32_t)(acc * BN + c * 32), v);
#pragma unroll
          for (int j = 0; j < 32; ++j) z[c * 32 + j] = fmaf(v[j], kUntruncate, z[c * 32 + j]);
        }
        tc_fence_before();
        mbar_arrive(tempty + acc);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) break;
      const int64_t tl = (!kTopk && live) ? (int64_t)a.targets[row] - col0 : -1;  // the target's place in this half
      TopkCursor cur;
      if constexpr (kTopk) {
        cur.open(a.topk, row, live, nb);
        cur.skip_to(col0);
      }
      // The maximum is kept of the unscaled values; exponents are differences to
      // it first, exact next to the maximum, then one product with scale log2 e.
      float m = -INFINITY, sum = 0.f, tz = 0.f;
      const float cexp = a.scale * kLog2e;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t cb = col0 + c * 32;
        float* v = z + c * 32;
        if constexpr (!std::is_void<TB>::value) {
          float b[32];
          load_bias32<TB>(a.bias, cb, a.V, b);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += b[j];
        }
        if (cb + 32 > a.V) {
          const int left = (int)(a.V - cb);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : -INFINITY;
        }
        if constexpr (kTopk) {
          int p;
          const uint32_t bits = cur.take(cb, p);
          if (__any_sync(0xffffffffu, bits != 0u)) {
            float* zo = a.topk.z + row * a.topk.K;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if ((bits >> j) & 1u) {
                zo[p + __popc(bits & ((1u << j) - 1u))] = v[j] * a.scale;
                v[j] = -INFINITY;
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
        for (int j = 1; j < 32; ++j) mc = fmaxf(mc, v[j]);
        const float nm = fmaxf(m, mc);
        if (nm != -INFINITY) {
          float part = 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) part += ex2((v[j] - nm) * cexp);
          sum = sum * ex2((m - nm) * cexp) + part;
          m = nm;
        }
      }
      if (live) {
        if (col0 < a.V) {
          const int64_t idx = (col0 / 128) * a.N + row;
          a.part_m[idx] = m * a.scale;
          a.part_s[idx] = sum;
        }
        if constexpr (!kTopk)
          if (tl >= 0 && tl < 128 && col0 + tl < a.V) a.tgt[row] = tz * a.scale;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename TB, bool kTopk>
cudaError_t logits_launch(const FwdArgs& f, cudaStream_t s) {
  const bool bf16 = f.dtype == CCE_BF16;
  CUtensorMap tmA, tmB;
  if (!make_tmap(&tmA, f.e, bf16, f.D, f.N, f.D, BK, BM)) return cudaErrorInvalidValue;
  if (!make_tmap(&tmB, f.c, bf16, f.D, f.V, f.D, BK, BN)) return cudaErrorInvalidValue;
  const LogitsArgs<TB> a{f.rows, f.targets, f.bias, f.part_m, f.part_s, f.tgt, f.N, f.V, (int)ceil_div(f.V, BN),
                         (int)ceil_div(f.D, BK), raster_group(f.N * f.D * 2), f.scale, f.topk};
  auto kern = tc_logits_kernel<TB, kTopk>;
  static std::atomic<unsigned long long> attr_ctx[64];
  cudaError_t err = ensure_smem_attr(kern, kLgSmem, attr_ctx);
  if (err != cudaSuccess) return err;
  const int64_t tiles = ceil_div(f.N, BM) * a.num_n;
  const int grid = tiles < num_sms() ? (int)tiles : num_sms();
  kern<<<grid, kLgThreads, kLgSmem, s>>>(tmA, tmB, a, instr_desc(BM, BN, bf16, false, false));
  return launched();
}

template <typename TB>
cudaError_t logits_dispatch(const FwdArgs& f, cudaStream_t s) {
  return f.topk.sid ? logits_launch<TB, true>(f, s) : logits_launch<TB, false>(f, s);
}
