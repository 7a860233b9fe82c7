// Internal launch interface between the C-ABI plan layer (plan.cpp) and the
// kernel families.  Nothing here crosses the library boundary.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "ask_types.h"

namespace askb {

// ---- family E: fused elementwise -------------------------------------------
constexpr int kEwThreads = 256;

enum EwSpec : int {
  EW_GENERIC = 0,
  EW_CFG1,
  EW_CFG5B,
  EW_SOFTMAX_NORM_F16,
  EW_SOFTMAX_NORM_BF16,
  EW_NUM_SPECS
};

// Division by a run-time invariant divisor d with a multiply-high and shifts
// (Granlund & Montgomery, "Division by Invariant Integers using
// Multiplication", PLDI 1994, unsigned case): for dividends below 2^32,
//   t = mulhi32(m, n); q = (t + ((n - t) >> s1)) >> s2
// with l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1, s1 = min(l, 1),
// s2 = max(l - 1, 0).  `wide` falls back to 64-bit division.
struct U32Div {
  uint64_t d;
  uint32_t m, s1, s2, wide;
};

struct EwArgs {
  const void* in[kMaxIn];
  void* out[kMaxOut];
  uint64_t count;
  U32Div inner;  // IM_OUTER / IM_INNER divisor
};

inline U32Div make_u32div(uint64_t d, uint64_t max_dividend) {
  U32Div q{d ? d : 1, 0, 0, 0, 1};
  if (d == 0 || d > 0xffffffffull || max_dividend > 0xffffffffull) return q;
  uint32_t l = 0;
  while ((uint64_t(1) << l) < d) ++l;
  const unsigned __int128 num = ((unsigned __int128)1 << 32) * ((unsigned __int128)((uint64_t(1) << l) - d));
  q.m = uint32_t(uint64_t(num / d) + 1);
  q.s1 = l < 1 ? l : 1;
  q.s2 = l > 1 ? l - 1 : 0;
  q.wide = 0;
  return q;
}

bool ew_spec_program(int spec, Program* out);
cudaError_t ew_occupancy(int spec, int* blocks_per_sm);
cudaError_t ew_launch(int spec, const Program& prog, const EwArgs& args, int aligned, int grid, cudaStream_t stream);

// ---- family R/T: map-reduce over [outer, extent, inner] ------------------------
constexpr int kRedThreads = 256;

enum RedSpec : int {
  RED_GENERIC = 0,
  RED_ROWSTATS_F32,      // cfg2: sum, max, min, argmax of f32 rows
  RED_GLOBAL_F32,        // cfg5a: sum, min, argmin of f32
  RED_SOFTMAX_MAX_F16,   // cfg3 step 0: max of cast(x, f32)
  RED_SOFTMAX_MAX_BF16,
  RED_SOFTMAX_SUM_F16,   // cfg3 step 1: sum of exp(cast(x) - m)
  RED_SOFTMAX_SUM_BF16,
  RED_NUM_SPECS
};

struct RedArgs {
  const void* in[kMaxIn];
  void* out[kMaxReductions];
  uint64_t outer, extent, inner;
  uint64_t index_base;   // added to arg-reduction indices (global offset of a shard)
  uint8_t n_red;
  uint8_t red_op[kMaxReductions];
  uint8_t red_src[kMaxReductions];   // which program output feeds each reduction
  uint8_t red_type[kMaxReductions];  // type of the reduced value (program output type)
};

// One partial accumulator as stored in scratch: value word + arg index.
struct RedPartial {
  uint64_t v;
  int64_t idx;
};

// Strategy chosen by the plan layer.
enum RedStrategy : int {
  RS_WARP_ROW = 0,   // inner == 1: one warp per output row, lanes stride the extent
  RS_COLUMN = 1,     // inner > 1: one thread per output column, loop over extent
  RS_SPLIT = 2,      // few outputs, huge extent: CTAs split the extent, partials in scratch
};

// Program and reduction list (all reductions fold program result 0) of a specialisation.
bool red_spec_program(int spec, Program* out, int* n_red, uint8_t* ops);
cudaError_t red_occupancy(int spec, int strategy, int* blocks_per_sm);
// RS_SPLIT writes grid * n_red partials to `scratch` and then combines them
// (second kernel) into the outputs, or, when `partials_out` is non-null, into
// one per-launch record per reduction (sharded plans combine those across ranks).
cudaError_t red_launch(int spec, int strategy, const Program& prog, const RedArgs& args, int aligned, int grid,
                       void* scratch, RedPartial* partials_out, cudaStream_t stream);
// Combine `n` records per reduction laid out [n][n_red] into the outputs.
cudaError_t red_combine_records(const RedArgs& args, const RedPartial* records, int n, cudaStream_t stream);
// Cross-GPU exchange of a sharded 0-D reduction's records over peer memory
// (one CTA): this rank's record `mine` (n_red records) is stored into slot
// `rank` of every rank's inbox (inboxes[r], device pointers valid on this
// device: the peers' inboxes are IPC mappings), each flag is raised with a
// release store, the rank waits (bounded by timeout_ns) for every rank's flag,
// and the records are folded in rank order into the outputs.  On a timeout the
// outputs are left as they were and the inbox's status word is set to 1.
constexpr int kExchangeMaxRanks = 64;
constexpr size_t kInboxRecordsBytes = size_t(2) * kExchangeMaxRanks * kMaxReductions * sizeof(RedPartial);
constexpr size_t kInboxFlagsOffset = kInboxRecordsBytes;                       // uint64 per rank
constexpr size_t kInboxSeqOffset = kInboxFlagsOffset + kExchangeMaxRanks * 8;  // uint64 epoch
constexpr size_t kInboxStatusOffset = kInboxSeqOffset + 8;                     // uint32, 0 = ok
constexpr size_t kInboxBytes = kInboxStatusOffset + 8;
cudaError_t red_exchange_combine(const RedArgs& args, const RedPartial* mine, void* const* inboxes, int nranks,
                                 int rank, uint64_t timeout_ns, cudaStream_t stream);
size_t red_split_scratch_bytes(int grid, int n_red);
// RS_COLUMN with few outputs: grid.y = chunks of the extent, one partial
// record per (output, chunk) in scratch, then a combine in chunk order.
cudaError_t red_column_chunks_launch(const Program& prog, const RedArgs& args, int grid, int chunks, void* scratch,
                                     cudaStream_t stream);
size_t red_column_chunks_scratch_bytes(uint64_t n_outputs, int chunks, int n_red);

// ---- family G / X: gather and scatter_add over [outer, D, inner] ------------------
struct IndexArgs {
  const void* table;     // gather: params; scatter: updates
  const void* index;
  void* out;
  const void* base;      // scatter: base tensor for the fused pre-copy (may equal out)
  uint64_t outer, dim, inner, n;  // params/base [outer, dim, inner]; index [n]
  int elem_type, index_type;
};
cudaError_t gather_launch(const IndexArgs& a, int aligned, int grid, cudaStream_t stream);
// `scratch` (scatter_sorted_scratch_bytes) enables the sorted path when
// scatter_sorted_ok holds; without it the element-atomic path runs.
cudaError_t scatter_add_launch(const IndexArgs& a, int aligned, int grid, void* scratch, int sms, cudaStream_t stream);
bool scatter_sorted_ok(const IndexArgs& a);
size_t scatter_sorted_scratch_bytes(const IndexArgs& a);
cudaError_t scatter_sorted_launch(const IndexArgs& a, void* scratch, int sms, cudaStream_t stream);

// ---- input synthesis (Philox4x32-10) -------------------------------------------------
enum GenKind : int { GEN_UNIFORM_F32 = 0, GEN_NORMAL_F32, GEN_NORMAL_F16, GEN_NORMAL_BF16, GEN_I32, GEN_ZIPF_I64, GEN_ZIPF_I32 };
// Elementwise steps with general index maps (IM_VIEW ports) or coordinate
// instructions: the runtime-program interpreter with per-element coordinates.
struct ViewSet {
  int rank;
  uint64_t shape[kMaxRank];
  PortView port[kMaxIn];
};
cudaError_t ew_view_launch(const Program& prog, const EwArgs& args, const ViewSet& views, int grid,
                           cudaStream_t stream);
int ew_view_occupancy();
// Reductions whose prologue reads IM_VIEW ports or coordinates: a warp per
// output over the [outer, extent, inner] domain of the iteration shape.
cudaError_t red_view_launch(const Program& prog, const RedArgs& a, const ViewSet& views, int grid,
                            cudaStream_t stream);
int red_view_occupancy();

// Family S: the three-step softmax plan fused (softmax_kernels.cu).  x and y
// are [rows, cols] f16/bf16 (16-byte aligned), m and s are [rows] f32.  The
// same row kernel also runs each step of the plan on its own (a reduce plan
// matched to ProgSoftmaxMax / ProgSoftmaxSum, an elementwise plan matched to
// ProgSoftmaxNorm): SM_STEP_MAX writes m only, SM_STEP_SUM reads m (m_in) and
// writes s only, SM_STEP_NORM reads m and s (m_in, s_in) and writes y only.
enum SoftmaxMode { SM_FUSED = 0, SM_STEP_MAX = 1, SM_STEP_SUM = 2, SM_STEP_NORM = 3 };
struct SoftmaxArgs {
  const void* x;
  float* m;
  float* s;
  void* y;
  const float* m_in;  // SM_STEP_SUM, SM_STEP_NORM
  const float* s_in;  // SM_STEP_NORM
  uint64_t rows, cols;
  int type;  // kF16 or kBF16
  int mode;  // SoftmaxMode
};
// 16-byte vectors each thread of a row's CTA holds, or 0 when cols has no
// fused kernel (cols must be a multiple of 256, at most 32768).
int softmax_vectors_per_thread(uint64_t cols);
cudaError_t softmax_rows_launch(const SoftmaxArgs& a, int sms, cudaStream_t stream);
// The grid softmax_rows_launch uses for `a` (SMs x resident CTAs, at most
// one CTA per row); needs the device current.
int softmax_rows_grid(const SoftmaxArgs& a, int sms);

// ---- training-block operators: dropout, block norms, bucketed-bias softmax -------------
// One dropout site: elements whose random word is below `threshold` =
// floor(p * 2^32) are dropped, the others scaled by `scale` = 1 / (1 - p).
struct DropSite {
  uint32_t on, threshold, stream;
  float scale;
};

// y = dropout(x) (+ residual), `count` contiguous elements (dropout_kernels.cu).
struct DropoutArgs {
  const void* x;
  const void* residual;  // null: none
  const int64_t* seed;   // {seed, offset} on the device
  void* y;
  uint64_t count;
  int type;
  DropSite drop;
};
cudaError_t dropout_launch(const DropoutArgs& a, int grid, cudaStream_t stream);
cudaError_t dropout_occupancy(int type, bool residual, int* blocks_per_sm);
constexpr int kDropThreads = 256;

// How a row's threads are laid out: see row_team.cuh.
struct TeamShape {
  int warp_teams;  // lanes of a warp that take a row (4 to 32), 0: the whole CTA or cluster
  int threads;     // of a CTA
  int team_threads;  // of a row's team within a CTA, where it is whole warps
  int ctas;        // of a row's cluster (1: no cluster)
  int elems;       // row elements a thread holds
};

// Block norms (norm_rows.cuh).  Forward: h = alpha x + D(gate * N_post(y)),
// u = N_pre(h); gradient: see the kernel.  x, y, h, u and the gradients to
// them are [rows, cols] of `type`; weights, biases [cols] and gate
// [groups, cols] of `ptype`; statistics [rows, 1 or 2] and the gradients to
// the parameters f32.
struct NormArgs {
  const void *x, *y, *w_post, *b_post, *gate, *w_pre, *b_pre;
  const int64_t* seed;
  void *h, *u;
  float *stats_post, *stats_pre;
  // gradient
  const void *dh, *du, *h_in;
  const float *stats_post_in, *stats_pre_in;
  void *dx, *dy;
  float *dw_post, *db_post, *dgate, *dw_pre, *db_pre;
  float* partial;  // [sum kinds][groups * chunks][cols]
  uint64_t rows, rows_per_group;
  uint32_t cols, groups, chunks;  // chunks of a group's rows, one CTA or cluster each (gradient)
  float alpha, eps;
  int type, ptype;
  int branch, post, pre, layer, bias, gated;
  // Rows begin at `classes` different places of a 16-byte unit (a power of two; 1
  // too where they are not read as cut units).
  // `spread` neighbouring CTAs (or clusters) share a stretch of rows, so that each
  // team's rows begin at one of them.
  uint32_t classes, spread;
  DropSite drop;
  TeamShape shape;
};
constexpr int kNormMaxCols = 32768;
constexpr int kNormJoinThreads = 16;  // that join one column's sums (gradient)
void norm_layout(NormArgs* a, bool grad);  // sets shape and classes
// How rows are read: as whole 16-byte units; as the units of the aligned tensor,
// cut at the rows' ends; else f32 by words and 16-bit types from anywhere.
enum NormFit { NORM_UNITS = 0, NORM_CUT = 1, NORM_WORDS = 2, NORM_ANYWHERE = 3 };
// Row sums the gradient keeps for each column: of B*yhat, B, du*hhat, du.
struct NormSums {
  bool t, s, p, q;
  int count() const { return int(t) + int(s) + int(p) + int(q); }
};
NormSums norm_sums(const NormArgs& a);
// Resident CTAs an SM, and the dynamic shared memory of one.
cudaError_t norm_occupancy(const NormArgs& a, NormFit fit, int* blocks_per_sm, unsigned* shared_bytes);
cudaError_t norm_grad_occupancy(const NormArgs& a, NormFit fit, int* blocks_per_sm, unsigned* shared_bytes);
cudaError_t norm_launch(const NormArgs& a, NormFit fit, int grid, cudaStream_t stream);
cudaError_t norm_grad_launch(const NormArgs& a, NormFit fit, cudaStream_t stream);
// Rows a CTA works on at once.
inline int team_count(const TeamShape& s) { return s.threads / (s.warp_teams ? s.warp_teams : s.team_threads); }

// Softmax over biased scores (bias_softmax.cuh).  s, p, dp, ds are
// [batch, heads, queries, keys] of `type`, table [buckets, heads] of
// `table_type`, lengths and offsets i32 [batch] (null: all keys, 0), lse
// [batch, heads, queries] f32.
constexpr int kBiasMaxThresholds = 255;
constexpr int kBiasMaxDistance = 4096;
constexpr uint64_t kBiasMaxKeys = 131072;
constexpr int kBiasMaxThreads = 512;  // of a CTA
constexpr int kBiasJoinThreads = 32;  // that join one entry of the table's gradient
struct BiasSoftmaxArgs {
  const void *s, *dp, *table;
  const float* lse_in;
  const int *lengths, *offsets;
  const int64_t* seed;
  void* out;       // p, or ds
  float* lse;      // forward
  float* dtable;   // gradient, [buckets, heads]
  float* partial;  // gradient: [heads * chunks * ctas][buckets]
  uint64_t batch, queries;
  uint64_t whole_rows;  // rows below this one may be read by whole units: those end inside the tensor
  uint32_t heads, keys, chunks;  // chunks of a head's (batch, query) pairs
  uint32_t buckets;
  float scale;
  int type, table_type;
  int causal, bidirectional, aligned;
  int n_thresholds;
  int thresholds[kBiasMaxThresholds];  // not falling; the bucket of a distance n is the number of them <= n
  DropSite drop;
  TeamShape shape;
  uint32_t ring_rows, window_copies, shared_bytes;  // rows in flight (1 or 2); the window's copies (0 or 1); of a CTA
};
TeamShape bias_softmax_shape(uint64_t keys, uint64_t rows, int type, bool grad, int sms);
// Threads of a CTA as the windows in shared memory allow, and those bytes.
void bias_softmax_shared(BiasSoftmaxArgs* a, bool grad);
cudaError_t bias_softmax_occupancy(const BiasSoftmaxArgs& a, int* blocks_per_sm);
cudaError_t bias_softmax_grad_occupancy(const BiasSoftmaxArgs& a, int* blocks_per_sm);
cudaError_t bias_softmax_launch(const BiasSoftmaxArgs& a, cudaStream_t stream);
cudaError_t bias_softmax_grad_launch(const BiasSoftmaxArgs& a, cudaStream_t stream);

cudaError_t gen_launch(int kind, uint64_t seed, uint32_t stream_id, uint64_t offset, uint64_t count, double p0,
                       double p1, const double* zipf_cdf, uint64_t zipf_n, void* dst, cudaStream_t stream);

}  // namespace askb
