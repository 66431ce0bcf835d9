// Internal launch interface between the C-ABI layer (cce_abi.cu) and the
// kernel translation units.  All launchers enqueue on `stream` and return the
// cudaError_t of the launch.
#pragma once

#include "common.cuh"
#include "peer.cuh"
#include "schedule.cuh"

namespace cce {

using tc::SlabPlan;

// Counts one kernel launch (cce_launch_count) and returns cudaGetLastError().
cudaError_t launched();

// Records `msg` as this thread's cce_last_error() and returns `code`.
int report_error(int code, const char* msg);

// Process-unique id of the CUDA context current on this thread (cuCtxGetId);
// *id = 0 when no context is current yet.  False if the driver calls fail.
// Per-context host state (device addresses of symbols, streams) is keyed by
// it: device ordinals are not enough once a host runs its own driver-API
// context or resets a device.
bool current_context_id(unsigned long long* id);

// Rows that count, moved to the front in order (rows_kernels.cu): their number,
// the batch row of each packed row, the packed row of each batch row (-1: left
// out), the packed rows' targets (nullptr: none).
struct RowsView {
  int32_t* count;
  int32_t* row_of;
  int32_t* pos;
  int32_t* targets;
};

// Per packed row up to K listed columns: sid[row][K] sorted and distinct,
// start[row][tiles1] the first entry of every kTopkTile-column tile (the last:
// the number of entries), z[row][K] a value per entry.
constexpr int kTopkTile = 128;
struct TopkView {
  const int32_t* sid = nullptr;
  const uint16_t* start = nullptr;
  float* z = nullptr;
  int K = 0, tiles1 = 0;
};

// The cotangent d of a batch row's log-probability or loss: factor * up (per row,
// or one for all), times weight[0].
struct Cotangent {
  const float* up;
  const float* weight;  // nullptr: 1
  float factor;
  int per_row;
#ifdef __CUDACC__
  __device__ __forceinline__ float of(int64_t packed, const int32_t* row_of) const {
    return up[per_row ? row_of[packed] : 0] * (weight ? weight[0] * factor : factor);
  }
#endif
};

// The power of two that a packed row's float16 dlogits are in units of.
struct RowScale {
  const float* s;  // [N], or one for all; nullptr: 1
  int per_row;
#ifdef __CUDACC__
  __device__ __forceinline__ float of(int64_t packed) const { return s ? s[per_row ? packed : 0] : 1.f; }
#endif
};

// GEMMs over a batch's packed rows (tc_rows.cuh), 16-bit operands; dtype CCE_F32:
// float32 operands as two float16 parts, x = (hi + lo / kLoUnits) / s[0] (e, c and
// e_lo, c_lo; se, sc: {s, 1 / s} on the device).
constexpr float kLoUnits = 2048.f;
struct RowsGemmArgs {
  const void *e, *e_lo;          // [N][Dk] packed rows, zeros behind the count
  const void *c, *c_lo;          // [V][Dk]
  const float *se, *sc;
  const void* bias;              // [V] or nullptr
  int bias_dtype, dtype;
  RowsView R;
  int64_t N, V, Dk, Dout;        // Dk: operands' width (a multiple of 8); Dout: the gradients'
                                 // (of 8, float32 of 4); their columns behind D are zeros
  int64_t vc0, vc_len;           // vocabulary rows of this call
  float scale_z;                 // logits = scale_z (e c^T + bias)
  TopkView topk;                 // the rows' listed columns (sid == nullptr: none)
  // row statistics
  float *part_m, *part_s, *tgt;  // [ceil(V / 128)][N] twice, [N]
  // dlogits and gradients
  const float *lse, *A;          // A: distillation
  Cotangent up;
  RowScale scale;                // float16 dlogits hold w / s of their row
  // grad_c: e with the rows' scales folded in, in units of max_s (the largest of them); se: its scale
  const void *ec, *ec_lo;
  const float *max_s, *sec;
  void *dl, *dl_lo;              // [N][vc_ld] 16-bit
  int64_t vc_ld;
  float* bias_part;              // [ceil(N / 32)][vc_ld] column sums of dlogits (those of the row tiles that
                                 // count are written and read), or nullptr
};

struct FwdArgs {
  const void* e;
  const void* c;
  const void* bias;
  int bias_dtype;
  const int32_t* targets;
  int64_t N, D, V, v_offset;
  int dtype;
  float* tile_max;  // [ceil(V / kStatTile)][N]: row max over each statistics tile (filter input)
  float* part_m;    // [P][N] (workspace): row max over each kernel tile, P = ceil(V / lse_tile)
  float* part_s;    // [P][N] (workspace): row sum of exp(logit - part_m) over the same columns
  float* tgt;       // [N]
};

struct BwdChunkArgs {
  const void* e;
  const void* c;         // row 0 of this call's c (the dense head; nullptr for a quantised one)
  const void* c_chunk;   // row vc0 of c: the chunk's vc_len rows (the dequantised chunk buffer
                         // for a quantised head); the chunk kernels read c through it
  const void* bias;
  int bias_dtype;
  const int32_t* targets;
  const float* lse;
  const float* d_nll;
  const uint8_t* keep;   // [nRb][nVt] block mask
  const uint32_t* keep_t;  // [ceil(V/128)][keep_t_ld] words: bit r of row m = a kept block of
                           // row block r in the 128 vocabulary columns of m (grad_c's M tiles)
  int64_t keep_t_ld;
  int64_t N, D, V, v_offset;
  int dtype;
  int64_t vc0;           // first local vocab row of the chunk
  int64_t vc_len;        // rows in the chunk
  int64_t vc_ld;         // row stride of the dlogits buffer (elements)
  void* dlogits;         // [N][vc_ld], fp32 (SIMT path) or 16-bit (tensor-core path)
  float* grad_bias;      // [V] fp32 or nullptr
  int* counters;         // 4 zeroed counters of this chunk (dlogits, grad_e, grad_c tile claims; the
                         // dlogits live-tile count) or nullptr
  const float* scale;    // fp16 tensor-core path: {s, 1/s} with s = 2^ceil(log2 max|d_nll|); else nullptr
  const int* dl_list = nullptr;  // the chunk's live dlogits tiles (tc_dlogits_lists), count in counters[3]
};

// ---- auxiliary kernels (aux_kernels.cu) ----
// (max, sum-exp) pairs, row p at part_max + p * ld (part_sum == nullptr: the
// entries are LSEs, i.e. pairs with sum 1)
cudaError_t launch_lse_combine(const float* part_max, const float* part_sum, const float* part_tgt,
                               int64_t P, int64_t N, int64_t ld, float* lse, float* tgt, float* nll,
                               cudaStream_t stream);
cudaError_t launch_block_mask(const float* tile_max, const float* lse, const int32_t* targets,
                              const float* d_nll, int64_t N, int64_t V, int64_t v_offset,
                              float log_eps, bool no_filter, uint8_t* keep, uint32_t* keep_t,
                              int64_t keep_t_ld, int64_t* skip_stats, cudaStream_t stream);
cudaError_t launch_cast_f32(const float* src, void* dst, int dtype, int64_t n, cudaStream_t stream);
// out[r][j] = scales[r][j / group] * q[r][j] + biases[r][j / group]  (cce_dequantize)
cudaError_t launch_dequantize(const uint32_t* wq, const void* scales, const void* biases, int scale_dtype,
                              int64_t rows, int64_t D, int group, int bits, int out_dtype, void* out,
                              cudaStream_t stream);
// dst[i] = a[i] + b[i], written in dtype (CCE_F32 / F16 / BF16)
cudaError_t launch_sum2_f32(const float* a, const float* b, void* dst, int dtype, int64_t n, cudaStream_t stream);
// out[0] = s = the power of two >= max |x| (1 if all zero), out[1] = 1 / s
cudaError_t launch_pow2_absmax(const float* x, int64_t n, float* out, cudaStream_t stream);
cudaError_t launch_fill_f32(float* dst, float v, int64_t n, cudaStream_t stream);

// ---- rows of a batch, distillation (rows_kernels.cu) ----
struct DistillSum {
  double loss;
  int32_t n;
};
// Row lists of the batch; mask_out and per_row_out (0 for rows left out) nullable;
// tgt: a value per packed row, zeroed (with targets); words: two, zeroed, nullable.
cudaError_t launch_rows_pack(int64_t N, const void* targets, int target_bytes, int64_t ignore_index, int has_ignore,
                             const uint8_t* mask, const RowsView& R, uint8_t* mask_out, float* per_row_out, float* tgt,
                             uint32_t* words, cudaStream_t stream);
// 16-bit rows: dst[i] = src[row_of[i]] (R; zeros behind the count), or src[i] (R == nullptr),
// `cols` values each, zeros up to dst_ld; word (zeroed, nullable): float16 bits of the largest finite |value|
cudaError_t launch_rows_copy(const void* src, int64_t rows, int64_t cols, int64_t src_ld, const RowsView* R, void* dst,
                             int64_t dst_ld, uint32_t* word, cudaStream_t stream);
// lse (packed rows) and logp (batch rows) from P partials
cudaError_t launch_rows_logp(const float* part_m, const float* part_s, int64_t P, int64_t N, const RowsView& R,
                             const float* tgt, float* lse, float* logp, cudaStream_t stream);
cudaError_t launch_topk_prep(const void* ids, int id_bytes, const float* logp, int64_t N, int64_t V, int K, double T,
                             int tail, const RowsView& R, const TopkView& topk, float* p, float* rest,
                             cudaStream_t stream);
int64_t distill_blocks(int64_t N);  // entries of `sums`
cudaError_t launch_distill_rows(const float* part_m, const float* part_s, int64_t P, int64_t N, int64_t V,
                                const RowsView& R, const TopkView& topk, const float* p, const float* rest,
                                int reduction, float* lse_rest, float* A, float* whole, DistillSum* sums, float* loss,
                                float* weight, cudaStream_t stream);
// out[n] = sum over the K splits' slabs (rows of ld values) of row pos[n], in order; 0 where pos[n] < 0
cudaError_t launch_rows_scatter(const float* slabs, const SlabPlan& plan, int64_t ld, const RowsView& R, int64_t N,
                                int64_t D, int dtype, void* out, cudaStream_t stream);
// A row's scale: the power of two >= |d| whole (whole nullptr: 1; below 1: 1) times 2^-14, into
// rows[N] where the cotangents are per row; max_s: the largest (and every row's, where they are not).
cudaError_t launch_rows_scale(const Cotangent& up, const float* whole, const RowsView& R, float* rows, float* max_s,
                              cudaStream_t stream);
// e's packed rows times rows / max_s, as one float16 value (lo nullptr; scale = {s, 1 / s} of the result, *word:
// the largest |e|) or two parts (in their own scale): what grad_c multiplies float16 dlogits of several scales by.
cudaError_t launch_rows_fold(const void* e, const void* e_lo, int64_t N, int64_t Dk, const RowsView& R,
                             const float* rows, const float* max_s, const uint32_t* word, float* scale, void* out,
                             void* out_lo, cudaStream_t stream);
// largest |x| of the rows (those of R, if given) as the bits of a float, into *word (zeroed)
cudaError_t launch_absmax(const float* x, int64_t rows, int64_t D, const RowsView* R, uint32_t* word,
                          cudaStream_t stream);
// x -> hi, lo [rows][Dp] and scale = {s, 1 / s}; R: the packed rows of x, zeros behind their count
cudaError_t launch_split(const float* x, int64_t rows, int64_t D, int64_t Dp, const RowsView* R, const uint32_t* word,
                         float* scale, void* hi, void* lo, cudaStream_t stream);
// column sums part[parts][ld] of 32 packed rows each -> out[cols]
cudaError_t launch_bias_sum(const float* part, int64_t parts, const RowsView& R, int64_t ld, int64_t cols, float* out,
                            cudaStream_t stream);

// ---- SIMT kernels (simt_kernels.cu): any dtype, any shape ----
cudaError_t simt_forward(const FwdArgs& a, cudaStream_t stream);
// vocabulary columns per LSE partial of simt_forward / tc_forward
constexpr int64_t kSimtLseTile = 128;
constexpr int64_t kTcLseTile = 256;
cudaError_t simt_dlogits(const BwdChunkArgs& a, cudaStream_t stream);
// grad_e_acc[N, D] (+)= dl[N, vc_len] @ c[v_offset-local rows vc0.., D]; with
// splits > 1 the K range is split over that many partial slabs part[splits][N][D]
// (workspace), summed in split order
cudaError_t simt_grad_e(const BwdChunkArgs& a, float* grad_e_acc, bool accumulate, float* part, int splits,
                        cudaStream_t stream);
// K splits simt_grad_e uses for an N x D output over chunks of vc rows
int simt_grad_e_splits(int64_t N, int64_t D, int64_t vc);
// grad_c[vc0 .. vc0+vc_len, D] = dl^T @ e, written in dtype
cudaError_t simt_grad_c(const BwdChunkArgs& a, void* grad_c, cudaStream_t stream);

// ---- tcgen05 kernels (tc_kernels.cu): 16-bit dtypes, D % 8 == 0 ----
bool tc_supported(const void* e, const void* c, int64_t D, int dtype);
bool tc_backward_supported(const void* e, const void* c, int64_t D, int dtype);
// Reads (and optionally clears) the tensor-core kernels' device status word:
// 0 = ok, > 0 = code of a bounded wait that timed out, -1 = read failed.
int tc_read_status(bool reset);
// Executed MMA FLOPs per kernel kind (forward, dlogits, grad_e, grad_c) since
// the last reset; 0 = ok, -1 = read failed.
int tc_read_mma_flops(uint64_t* out4, bool reset);
cudaError_t tc_forward(const FwdArgs& a, cudaStream_t stream);
cudaError_t tc_dlogits(const BwdChunkArgs& a, cudaStream_t stream);
// Lists, per vocabulary chunk of vc rows, the dlogits work units with a kept
// block in schedule order: chunk ch's ids at lists + ch * tc_dlogits_list_len(N, vc),
// their count in counters[4 ch + 3] (zeroed before).  One block per chunk.
int64_t tc_dlogits_list_len(int64_t N, int64_t vc);
cudaError_t tc_dlogits_lists(const uint8_t* keep, int64_t N, int64_t D, int64_t V, int64_t vc, int* lists,
                             int* counters, cudaStream_t stream);
// acc2[2][N][D] fp32: each output tile's two K halves of this chunk are
// stored (accumulate = false) or added into slabs 0 and 1; grad_e is
// acc2[0] + acc2[1] after the last chunk (launch_sum2_f32).  With `push`
// (the last chunk of a vocabulary-sharded backward) each half, plus its slab
// when accumulating, goes to its rows' owner rank instead (peer.cuh).
struct PeerPush {
  peer::Peers peers;
  peer::Layout layout;
};
cudaError_t tc_grad_e(const BwdChunkArgs& a, float* acc2, bool accumulate, const PeerPush* push,
                      cudaStream_t stream);
cudaError_t tc_grad_c(const BwdChunkArgs& a, void* grad_c, cudaStream_t stream);
// one bounded pipeline wait that nothing satisfies: records `code` after limit_ns
cudaError_t tc_selftest_wait(uint64_t limit_ns, int code, cudaStream_t stream);

// ---- GEMMs over packed rows (tc_rows.cuh) ----
bool tc_available();  // the driver's tensor-map encoder was found
cudaError_t tc_logits(const RowsGemmArgs& a, cudaStream_t stream);
cudaError_t tc_dlogits_rows(const RowsGemmArgs& a, cudaStream_t stream);
// slabs[plan.cap 128][Dout] (+)= the K splits of dl c (fp32)
cudaError_t tc_grad_e_rows(const RowsGemmArgs& a, float* slabs, const SlabPlan& plan, bool accumulate,
                           cudaStream_t stream);
// grad_c rows [vc0, vc0 + vc_len) = dl^T e, row stride Dout
cudaError_t tc_grad_c_rows(const RowsGemmArgs& a, void* grad_c, cudaStream_t stream);

// ---- losses on per-token log-probabilities (token_loss.cu) ----
// Sequences: offsets cu[S + 1] into the N tokens, or (cu == nullptr) S rows of N / S tokens.
struct PolicyArgs {
  const void *logp, *old, *ref;  // [N] of dtype; old, ref nullable
  int dtype;
  const float* adv;              // [N] (adv_token) or [S]
  int adv_token;
  const uint8_t* mask;           // [N], nullable
  const int32_t* cu;
  int64_t N, S;
  int reduction;                 // CCE_REDUCE_*
  double clip_low, clip_high, dual_clip, kl_coef;
  float *loss, *stats, *coef, *weight;  // [1] or [N], [2], [N], [1 + S]
};
struct PreferenceArgs {
  const void *logp, *ref;        // [N] of dtype; ref nullable
  int dtype;
  const float* ref_seq;          // [2 pairs], nullable
  const uint8_t* mask;           // [N], nullable
  const int32_t* cu;             // S = 2 pairs
  int64_t N, pairs;
  int kind, reduction, by_length;  // CCE_PREF_*, CCE_REDUCE_*
  double beta, margin, smoothing;
  float *loss, *rewards, *coef;  // [1] or [pairs], [2 pairs], [2 pairs]
};
size_t token_loss_workspace_bytes(int64_t N, int64_t S);
cudaError_t policy_forward(const PolicyArgs& a, void* ws, cudaStream_t stream);
cudaError_t policy_backward(const float* coef, const float* weight, const float* up, int up_token, int reduction,
                            const int32_t* cu, int64_t N, int64_t S, int dtype, void* grad, cudaStream_t stream);
cudaError_t preference_forward(const PreferenceArgs& a, void* ws, cudaStream_t stream);
cudaError_t preference_backward(const float* coef, const float* up, int up_pair, const uint8_t* mask, const int32_t* cu,
                                int64_t N, int64_t pairs, int dtype, void* grad, cudaStream_t stream);

// ---- cross-rank grad_e exchange (peer.cu) ----
namespace peer {
// partial rows src[nslab][N][D] fp32 -> their owners' receive slots; raises `pushed`
cudaError_t launch_push(const Peers& P, const Layout& L, const float* src, int nslab, int64_t N, int64_t D,
                        cudaStream_t stream);
// reduce this rank's rows (nslot slots per source) into out (out_dtype) and the
// reduced area, then gather the other ranks' rows into out
cudaError_t launch_reduce_gather(const Peers& P, const Layout& L, int nslot, int64_t N, int64_t D, int out_dtype,
                                 void* out, uint64_t limit_ns, cudaStream_t stream);
// status word of the exchange kernels' bounded waits (0 = ok, -1 = read failed)
int read_status(bool reset);
}  // namespace peer

}  // namespace cce
