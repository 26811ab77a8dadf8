// finetune.inl -- host side of the fine-tuning operators (included at the end of trebi.hip): argument checks and launch
// shapes of the gradient norm (gradnorm.hip), the policy loss (policy.hip), the preference loss (pairs.hip) and the
// transition log-probability (transition.hip).  Nothing here allocates, synchronises or keeps state: tables and workspaces are the caller's.
#include "finetune.h"

namespace {

size_t al256(size_t n) { return (n + 255) / 256 * 256; }

// Elements of a chunk.  Up to 8 M elements each workgroup gets one of 4096, whose loads are all in flight at once (bfloat16,
// 4 M elements in 50 tensors, clipped in place: 9.2 us, with 16384 13.2; 2 M: 7.2, with 2048 8.2).  Larger sets: whole turns of a
// workgroup (256 threads x 8 loads of 16 bytes: 16384 16-bit or 8192 32-bit elements), at most about 8 chunks each, so that
// all end together (20 M: 24 us, with 4096 29; 400 M: 442, with 4096 461).
long long grad_chunk(long long total) {
  if (total <= 4096ll * GRAD_BLOCKS) return 4096;
  const long long per = (total + 8 * GRAD_BLOCKS - 1) / (8 * GRAD_BLOCKS);
  return std::min<long long>((per + 16383) / 16384 * 16384, 1 << 28);
}

int grad_totals(int n, const int64_t* numels, long long* total, long long* chunks) {
  if (n < 1 || !numels) return fail(TREBI_BAD_ARG, "at least one tensor is needed");
  *total = 0;
  for (int i = 0; i < n; ++i) {
    if (numels[i] < 0 || numels[i] > (1ll << 48)) return fail(TREBI_BAD_ARG, "tensor %d has a bad size", i);
    *total += numels[i];
  }
  const long long c = grad_chunk(*total);
  *chunks = 0;
  for (int i = 0; i < n; ++i) *chunks += (numels[i] + c - 1) / c;
  if (*chunks > 0x7fffffff) return fail(TREBI_UNSUPPORTED_CONFIG, "too many tensors for one set");
  return 0;
}

// From this many bytes on the 256 MB cache cannot hand a set from one kernel to the next: such sets are read (for the norm
// alone) and written past the caches.  Norm of 366 MB 59 us, through them 67; 976 MB 151 and 172; 244 MB: 42 both ways.
// Clipping 200 M bfloat16 into float32: 315 us, through them 353.
constexpr long long GRAD_STREAM = 256ll << 20;

int grad_args(trebi_ctx* ctx, const trebi_grad_set* set, const void* table, int norm_type, float grad_scale, void* ws,
              size_t ws_bytes, GradP* p) {
  if (!ctx || !set || !table || !ws) return fail(TREBI_BAD_ARG, "null argument");
  if (norm_type < 0 || norm_type > 2) return fail(TREBI_BAD_ARG, "norm_type must be 0 (two-norm), 1 (one-norm) or 2 (largest)");
  if (set->n_tensors < 1 || set->n_chunks < 0) return fail(TREBI_BAD_ARG, "the set was not filled");
  if (!(grad_scale >= 0.f)) return fail(TREBI_BAD_ARG, "grad_scale must not be negative");
  if (ws_bytes < trebi_grad_workspace_bytes(set))
    return fail(TREBI_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", ws_bytes, trebi_grad_workspace_bytes(set));
  p->chunks = (const GradChunk*)table;
  p->n_chunks = set->n_chunks;
  const int rounds = std::max(1, (set->n_chunks + GRAD_BLOCKS - 1) / GRAD_BLOCKS);    // the same number of chunks for every workgroup
  p->n_blocks = std::max(1, (set->n_chunks + rounds - 1) / rounds);
  p->one_each = set->n_chunks > 0 && set->n_chunks <= GRAD_BLOCKS && grad_chunk(set->total) <= 4096;
  p->norm_type = norm_type;
  p->grad_scale = grad_scale;
  p->part = (double*)ws;
  return 0;
}

int token_args(const trebi_token_desc& d, TokenP* t) {
  if (d.rows < 0 || d.len < 0 || d.rows > (1ll << 40) || d.len > (1ll << 40)) return fail(TREBI_BAD_SHAPE, "bad number of rows or tokens");
  if (d.packed) {
    if (!d.cu_seqlens) return fail(TREBI_BAD_ARG, "packed tokens need cu_seqlens");
    if (d.rows < 1) return fail(TREBI_BAD_SHAPE, "packed tokens need at least one sequence");
    if (d.lengths) return fail(TREBI_BAD_ARG, "lengths belong to padded rows");
    if (d.len > 0x7fffffff || d.rows > 0x7fffff00)
      return fail(TREBI_UNSUPPORTED_CONFIG, "cu_seqlens is 32-bit: at most 2^31 - 1 packed tokens, fewer sequences");
    if (d.mask && d.mask_col_stride != 1) return fail(TREBI_BAD_ARG, "a packed mask is contiguous");
  } else {
    if (d.cu_seqlens) return fail(TREBI_BAD_ARG, "cu_seqlens belongs to packed tokens");
    if (d.len > 0 && d.rows > (1ll << 46) / d.len) return fail(TREBI_BAD_SHAPE, "too many tokens");
  }
  t->rows = d.rows;
  t->len = d.len;
  t->n = d.packed ? d.len : d.rows * d.len;
  t->packed = d.packed ? 1 : 0;
  t->lengths = d.lengths;
  t->cu = d.cu_seqlens;
  t->mask = d.mask;
  t->mrs = d.mask_row_stride;
  t->mcs = d.mask_col_stride;
  return 0;
}

// One workgroup does it all up to 4096 tokens (at most 4 turns): calls of this size wait for their launches.  4096 float32 tokens
// with lengths, enqueued one by one: 13.6 us, with two launches 17.6 (replayed from a graph 10.8 and 8.6); 8192: 18.2 and 17.7 (18.3 and 8.7).
// policy workspace: partial counts, partial sums, a count for each row; a call of one workgroup without a mask needs none
constexpr long long SINGLE = 4096;
// Up to this many rows every workgroup adds their lengths up for itself, which saves a launch: 1024 x 1024 float32 with lengths
// 12.5 us against 14.3, 2048 x 1024 16.4 and 17.2, 4096 x 1024 25.3 and 23.0, 16384 x 1024 76 and 58.
constexpr long long COUNT_ROWS = 2048;
size_t policy_bytes(const trebi_token_desc& d) {
  if (!d.mask && d.rows >= 0 && d.rows <= SINGLE && d.len >= 0 && (d.packed || d.len <= SINGLE) && (d.packed ? d.len : d.rows * d.len) <= SINGLE) return 0;
  return al256(COUNT_BLOCKS * sizeof(NormPart)) + al256((LOSS_PARTS * LOSS_VALS + 1) * sizeof(double)) +
         (d.mask ? al256((size_t)d.rows * sizeof(int)) : 0);
}

constexpr int PAIR_BLOCKS = 2048;
// Rows are split over workgroups where whole pairs would leave the card idle: at most one pair a CU, and rows long enough to
// pay for the second read and the third launch.  float32: 24 pairs of 131072 tokens 23 us, whole 88; 24 x 16384 10 and 16; 100 x
// 16384 17.5 and 19; 250 x 16384 27, whole 23; 24 x 8192 10 both ways.  (Lengths on the device do not matter for the choice.)
int pair_splits(const trebi_token_desc& d) {
  const long long len = d.packed ? (d.len + d.rows - 1) / d.rows : d.len;
  if (d.rows > 512 || len <= 8192 || len < 64 * d.rows) return 0;
  return (int)std::max<long long>(1, std::min<long long>(PAIR_BLOCKS / d.rows, (len + 4095) / 4096));
}
// Threads of a pair.  A wave pays for its pairs' scalars (a few hundred instructions) whatever it holds: few pairs take a whole
// workgroup each, many pairs of short rows 16 threads.  bfloat16, us with 16 / 64 / 256 threads: 512 pairs of 60 tokens 7.7 / 8.2 /
// 7.9, of 500 11 / 8.1 / 7.8, of 2000 27 / 12 / 9.5; 2000 of 1000 18 / 13 / 18; 8000 of 200 12 / 19 / 39.
int pair_group(const trebi_token_desc& d) {
  const long long len = d.packed ? (d.len + d.rows - 1) / d.rows : d.len, pairs = d.rows / 2;
  if (len <= 128 || (pairs > 4096 && len <= 512)) return 16;
  return pairs > 1024 && len <= 4096 ? 64 : 256;
}
long long pair_blocks(const trebi_token_desc& d) {
  const int per = 256 / pair_group(d);
  return (d.rows / 2 + per - 1) / per;
}
// preference workspace: partial sums, the rows' parts; a call of one workgroup needs none
size_t pair_bytes(const trebi_token_desc& d) {
  if (d.rows < 2) return 0;
  const int s = pair_splits(d);
  if (!s && pair_blocks(d) == 1) return 0;
  return s ? al256((size_t)d.rows / 2 * 4 * sizeof(double)) + al256((size_t)d.rows * s * 2 * sizeof(double))
           : al256((size_t)pair_blocks(d) * 4 * sizeof(double));
}

}  // namespace

// ---------------------------------------------------------------------------------------------------------------
// global gradient norm
// ---------------------------------------------------------------------------------------------------------------
extern "C" size_t trebi_grad_set_bytes(int n_tensors, const int64_t* numels) {
  long long total, chunks;
  if (grad_totals(n_tensors, numels, &total, &chunks)) return 0;
  return al256((size_t)std::max<long long>(chunks, 1) * sizeof(GradChunk));
}

extern "C" int trebi_grad_set_fill(int n_tensors, const void* const* tensors, const int64_t* numels, const int* dtypes,
                                   void* host_table, size_t table_bytes, trebi_grad_set* out) {
  long long total, chunks;
  if (!tensors || !dtypes || !host_table || !out) return fail(TREBI_BAD_ARG, "null argument");
  if (int e = grad_totals(n_tensors, numels, &total, &chunks)) return e;
  if (table_bytes < trebi_grad_set_bytes(n_tensors, numels)) return fail(TREBI_WORKSPACE_TOO_SMALL, "table of %zu bytes", table_bytes);
  for (int i = 0; i < n_tensors; ++i) {
    if (dtypes[i] < 0 || dtypes[i] > 2) return fail(TREBI_BAD_ARG, "tensor %d has an unknown type %d", i, dtypes[i]);
    const size_t size = dtypes[i] == TREBI_F32 ? 4 : 2;
    if (numels[i] && (!tensors[i] || (uintptr_t)tensors[i] % size)) return fail(TREBI_BAD_ARG, "tensor %d is null or not aligned to its type", i);
  }
  // a byte of two tensors would be scaled twice, by two workgroups at once
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> span;
    for (int i = 0; i < n_tensors; ++i)
      if (numels[i] > 0) span.push_back({(uintptr_t)tensors[i], (uintptr_t)tensors[i] + (size_t)numels[i] * (dtypes[i] == TREBI_F32 ? 4 : 2)});
    std::sort(span.begin(), span.end());
    for (size_t i = 1; i < span.size(); ++i)
      if (span[i].first < span[i - 1].second) return fail(TREBI_BAD_ARG, "two of the tensors overlap (or one is given twice)");
  } catch (const std::exception& e) {
    return fail(TREBI_HIP_ERROR, "out of host memory: %s", e.what());
  }
  const long long c = grad_chunk(total);
  GradChunk* ch = (GradChunk*)host_table;
  *ch = GradChunk{nullptr, 0, 0, 0};                       // (a set of empty tensors)
  long long at = 0, bytes = 0;
  for (int i = 0; i < n_tensors; ++i) {
    const size_t size = dtypes[i] == TREBI_F32 ? 4 : 2;
    for (long long o = 0; o < numels[i]; o += c)
      *ch++ = GradChunk{(char*)tensors[i] + o * size, at + o, (int)std::min<long long>(c, numels[i] - o), dtypes[i]};
    at += numels[i];
    bytes += numels[i] * size;
  }
  out->n_tensors = n_tensors;
  out->n_chunks = (int)chunks;
  out->total = total;
  out->bytes = bytes;
  return 0;
}

extern "C" size_t trebi_grad_workspace_bytes(const trebi_grad_set* set) { return set ? GRAD_BLOCKS * sizeof(double) : 0; }

extern "C" int trebi_grad_norm(trebi_ctx* ctx, const trebi_grad_set* set, const void* table, int norm_type, float grad_scale,
                               float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  GradP p{};
  if (int e = grad_args(ctx, set, table, norm_type, grad_scale, workspace, workspace_bytes, &p)) return e;
  if (!norm_out) return fail(TREBI_BAD_ARG, "norm_out is null");
  p.norm_out = norm_out;
  p.stream_loads = set->bytes > GRAD_STREAM;
  ON_DEVICE(ctx);
  HIPCHK(launch_grad_partials(p, (hipStream_t)stream));
  HIPCHK(launch_grad_finish(p, nullptr, (hipStream_t)stream));
  return 0;
}

extern "C" int trebi_grad_clip(trebi_ctx* ctx, const trebi_grad_set* set, const void* table, int norm_type, float max_norm,
                               float grad_scale, float* out, float* norm_out, void* workspace, size_t workspace_bytes,
                               void* stream) {
  GradP p{};
  if (int e = grad_args(ctx, set, table, norm_type, grad_scale, workspace, workspace_bytes, &p)) return e;
  if (!(max_norm >= 0.f)) return fail(TREBI_BAD_ARG, "max_norm must not be negative");
  p.max_norm = max_norm;
  p.out = out;
  p.norm_out = norm_out;
  p.stream_stores = set->bytes + (out ? 4 * set->total : 0) > GRAD_STREAM;
  ON_DEVICE(ctx);
  HIPCHK(launch_grad_partials(p, (hipStream_t)stream));
  HIPCHK(launch_grad_scale(p, (hipStream_t)stream));
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------
// clipped policy loss
// ---------------------------------------------------------------------------------------------------------------
extern "C" size_t trebi_policy_loss_workspace_bytes(const trebi_token_desc* d) { return d ? policy_bytes(*d) : 0; }

extern "C" int trebi_policy_loss(trebi_ctx* ctx, const trebi_token_desc* tokens, const trebi_policy_loss_desc* d, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!ctx || !tokens || !d || (!workspace && policy_bytes(*tokens))) return fail(TREBI_BAD_ARG, "null argument");
  PolicyP p{};
  if (int e = token_args(*tokens, &p.tk)) return e;
  const bool empty = p.tk.n == 0;
  if (!d->stats || (!empty && (!d->logp || !d->advantages))) return fail(TREBI_BAD_ARG, "null argument");
  if (d->dtype < 0 || d->dtype > 2) return fail(TREBI_BAD_ARG, "unknown type %d", d->dtype);
  if (d->kl_kind < 1 || d->kl_kind > 3) return fail(TREBI_BAD_ARG, "kl_kind must be 1, 2 or 3");
  if (d->reduction < 0 || d->reduction > 2) return fail(TREBI_BAD_ARG, "reduction must be 0 (token), 1 (sequence) or 2 (denominator)");
  if (!(d->clip_low >= 0.f) || !(d->clip_high >= 0.f)) return fail(TREBI_BAD_ARG, "clip ranges must not be negative");
  if (d->dual_clip != 0.f && !(d->dual_clip > 1.f)) return fail(TREBI_BAD_ARG, "dual_clip must be above 1 (or 0: off)");
  if (d->reduction == 1 && tokens->mask && tokens->len > 0x7fffffff)
    return fail(TREBI_UNSUPPORTED_CONFIG, "the mean over masked sequences counts at most 2^31 - 1 tokens a row");
  if (d->reduction == 2 && !(d->denominator > 0.0)) return fail(TREBI_BAD_ARG, "denominator must be positive");
  if (workspace_bytes < policy_bytes(*tokens)) return fail(TREBI_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes, policy_bytes(*tokens));
  p.lp = d->logp; p.old = d->logp_old; p.ref = d->logp_ref;
  p.lrs = d->logp_row_stride; p.lcs = d->logp_col_stride;
  p.ors = d->old_row_stride; p.ocs = d->old_col_stride;
  p.rrs = d->ref_row_stride; p.rcs = d->ref_col_stride;
  p.adv = d->advantages; p.ars = d->adv_row_stride; p.acs = d->adv_col_stride;
  p.grad = d->grad;
  // the borders in the log, in float64, of the float32 ranges that the caller gave; the ratio held there is 1 + range
  p.hi = std::log1p((double)d->clip_high);
  p.lo = d->clip_low < 1.f ? std::log1p(-(double)d->clip_low) : -INFINITY;
  p.dual = d->dual_clip > 1.f ? std::log((double)d->dual_clip) : INFINITY;
  p.fhi = (float)p.hi; p.flo = (float)p.lo; p.fdual = (float)p.dual;
  p.vhi = (float)(1.0 + (double)d->clip_high);
  p.vlo = (float)(1.0 - (double)d->clip_low);
  p.vdual = d->dual_clip;
  p.kl_coef = d->kl_coef; p.kl = d->kl_kind; p.mode = d->reduction; p.gscale = d->grad_scale;
  p.stats = d->stats;
  TokenP& t = p.tk;
  // Rows of one token are one row of tokens, to either mean, and that goes 16 bytes a thread instead of token by token (4 M
  // float32: 20 us, as rows 31; bfloat16 18 and 35)
  if (!t.packed && t.len == 1 && !t.lengths && (!t.mask || t.mrs == 1)) {
    t.len = t.rows;
    t.rows = 1;
    p.lcs = p.lrs; p.ocs = p.ors; p.rcs = p.rrs; t.mcs = t.mrs; p.acs = p.ars;
    if (p.mode == 1) p.mode = 0;
  }
  if (t.rows == 1 && p.mode == 1) p.mode = 0;                         // the mean over one sequence is the mean over its tokens
  const long long L = t.len;
  if (!t.packed && t.rows == 1) {                                     // strides that no step uses
    p.lrs = p.ors = p.rrs = t.mrs = L;
    if (p.acs) p.ars = L;
  }
  if (!t.packed && L == 1) {
    p.lcs = p.ocs = p.rcs = t.mcs = 1;
    p.acs = 0;
  }
  const bool flat_lp = t.packed ? p.lcs == 1 : p.lcs == 1 && p.lrs == L;
  const bool flat_old = !p.old || (t.packed ? p.ocs == 1 : p.ocs == 1 && p.ors == L);
  const bool flat_ref = !p.ref || (t.packed ? p.rcs == 1 : p.rcs == 1 && p.rrs == L);
  const bool flat_adv = p.acs == 0 || (t.packed ? p.acs == 1 : p.acs == 1 && p.ars == L);
  const bool flat_mask = !t.mask || (t.packed ? t.mcs == 1 : t.mcs == 1 && t.mrs == L);
  p.flat = flat_lp && flat_old && flat_ref && flat_adv && flat_mask;
  if (t.packed && !p.flat) return fail(TREBI_UNSUPPORTED_CONFIG, "packed tensors are contiguous");
  // rows shorter than the tokens of a thread (packed: than 8 on average) go token by token: these would lie in many rows
  const int pack = d->dtype == TREBI_F32 ? 4 : 8;
  if (t.packed ? t.n < 8 * t.rows : L < pack) p.flat = 0;
  const bool all = !t.packed && !t.lengths && !t.mask;
  if (p.mode == 2) p.fixed = 1.0 / d->denominator;
  else if (all && !empty) p.fixed = 1.0 / (double)(p.mode == 0 ? t.n : t.rows);
  char* w = (char*)workspace;
  p.np = (NormPart*)w; w += al256(COUNT_BLOCKS * sizeof(NormPart));
  p.part = (double*)w; w += al256((LOSS_PARTS * LOSS_VALS + 1) * sizeof(double));
  p.weight = p.part + LOSS_PARTS * LOSS_VALS;
  p.counts = t.mask && p.mode == 1 ? (int*)w : nullptr;
  hipStream_t st = (hipStream_t)stream;
  ON_DEVICE(ctx);
  const long long turn = 256 * pack, turns = (t.n + turn - 1) / turn;
  // as many workgroups as fit on the 256 CUs at once, so that none is left for a second round: 5 or (see the kernel) 4
  const long long most = t.packed || p.acs || (p.ref && p.kl == 3) ? 1024 : LOSS_PARTS;
  const long long per = t.n <= SINGLE ? std::max<long long>(turns, 1) : (turns + most - 1) / most;
  const int blocks = (int)((turns + per - 1) / per);
  p.per = per * turn;
  p.early = all || (t.packed && !t.mask) || per == 1;
  const bool told = t.packed && p.mode == 0 && !t.mask;               // the offsets say how many tokens there are
  if (!empty && !told && (p.counts || (p.fixed == 0.0 && (t.mask || t.rows > (blocks == 1 ? SINGLE : COUNT_ROWS))))) {
    HIPCHK(launch_token_counts(p, st));
  }
  if (!empty) HIPCHK(launch_policy(p, d->dtype, blocks, st));
  if (blocks == 1) return 0;
  HIPCHK(launch_policy_finish(p, blocks, st));
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------
// preference loss
// ---------------------------------------------------------------------------------------------------------------
extern "C" size_t trebi_preference_loss_workspace_bytes(const trebi_token_desc* d) { return d ? pair_bytes(*d) : 0; }

extern "C" int trebi_preference_loss(trebi_ctx* ctx, const trebi_token_desc* tokens, const trebi_preference_loss_desc* d,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  if (!ctx || !tokens || !d) return fail(TREBI_BAD_ARG, "null argument");
  PairP p{};
  if (int e = token_args(*tokens, &p.tk)) return e;
  if (p.tk.rows < 2 || p.tk.rows % 2) return fail(TREBI_BAD_SHAPE, "%lld rows: chosen and rejected rows come in pairs", (long long)p.tk.rows);
  if (!pair_splits(*tokens) && pair_blocks(*tokens) > 0xffffff) return fail(TREBI_UNSUPPORTED_CONFIG, "too many pairs for one call");
  if (!d->stats || !d->chosen_reward || !d->rejected_reward || (p.tk.n > 0 && !d->logp)) return fail(TREBI_BAD_ARG, "null argument");
  if (d->dtype < 0 || d->dtype > 2) return fail(TREBI_BAD_ARG, "unknown type %d", d->dtype);
  if (d->kind < 0 || d->kind > 2) return fail(TREBI_BAD_ARG, "kind must be 0 (sigmoid), 1 (hinge) or 2 (ipo)");
  if (!(d->beta > 0.f)) return fail(TREBI_BAD_ARG, "beta must be positive");
  if (!(d->label_smoothing >= 0.f) || !(d->label_smoothing < 0.5f)) return fail(TREBI_BAD_ARG, "label_smoothing must lie in [0, 0.5)");
  if (d->denominator < 0.0 || d->denominator != d->denominator) return fail(TREBI_BAD_ARG, "denominator must be positive (0: the number of pairs)");
  if (!workspace && pair_bytes(*tokens)) return fail(TREBI_BAD_ARG, "workspace is null");
  if (workspace_bytes < pair_bytes(*tokens)) return fail(TREBI_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes, pair_bytes(*tokens));
  p.pairs = p.tk.rows / 2;
  p.lp = d->logp; p.ref = d->logp_ref;
  p.lrs = d->logp_row_stride; p.lcs = d->logp_col_stride;
  p.rrs = d->ref_row_stride; p.rcs = d->ref_col_stride;
  if (p.tk.packed && (p.lcs != 1 || (p.ref && p.rcs != 1))) return fail(TREBI_UNSUPPORTED_CONFIG, "packed tensors are contiguous");
  p.weights = d->weights;
  p.grad = p.tk.n > 0 ? d->grad : nullptr;
  p.beta = d->beta; p.margin = d->margin; p.smooth = d->label_smoothing; p.gscale = d->grad_scale;
  p.inv_p = 1.0 / (d->denominator > 0.0 ? d->denominator : (double)p.pairs);
  p.kind = d->kind; p.average = d->average ? 1 : 0;
  p.rew_c = d->chosen_reward; p.rew_r = d->rejected_reward;
  p.stats = d->stats;
  p.part = (double*)workspace;
  p.splits = pair_splits(*tokens);
  p.rowpart = !p.splits ? nullptr : (double*)((char*)workspace + al256((size_t)p.pairs * 4 * sizeof(double)));
  hipStream_t st = (hipStream_t)stream;
  ON_DEVICE(ctx);
  if (p.splits) {
    p.nparts = (int)p.pairs;
    HIPCHK(launch_pairs_split(p, d->dtype, st));
  } else {
    p.group = pair_group(*tokens);
    p.nparts = (int)pair_blocks(*tokens);
    HIPCHK(launch_pairs_whole(p, d->dtype, st));
  }
  if (p.splits || p.nparts > 1) HIPCHK(launch_pairs_finish(p, st));
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------
// transition log-probability
// ---------------------------------------------------------------------------------------------------------------
static int transition_args(trebi_ctx* ctx, const trebi_transition_desc* d, const float* pred, const float* x, const float* x_prev,
                           const int64_t* t, int64_t B, TransP* p) {
  if (!ctx || !d) return fail(TREBI_BAD_ARG, "null argument");
  if (B < 0) return fail(TREBI_BAD_SHAPE, "negative batch");
  if (d->horizon < 1 || d->transition_dim < 1 || d->action_dim < 0 || d->observation_dim < 0 || d->n_timesteps < 1 ||
      d->action_dim + d->observation_dim > d->transition_dim || (long long)d->horizon * d->transition_dim > 1 << 28)
    return fail(TREBI_BAD_SHAPE, "inconsistent dimensions");
  if (B > 0 && (!pred || !x || !x_prev || !t)) return fail(TREBI_BAD_ARG, "null argument");
  if (!d->posterior_log_variance || !d->coef1 || !d->coef2) return fail(TREBI_BAD_ARG, "null schedule table");
  if ((d->sqrt_recip_alphas_cumprod == nullptr) != (d->sqrt_recipm1_alphas_cumprod == nullptr))
    return fail(TREBI_BAD_ARG, "sqrt_recip_alphas_cumprod and sqrt_recipm1_alphas_cumprod go together");
  if (d->n_cond < 0 || d->n_cond > 4) return fail(TREBI_UNSUPPORTED_CONFIG, "at most 4 conditioned timesteps are supported");
  const int H = d->horizon, D = d->transition_dim;
  p->B = B; p->H = H; p->D = D; p->T = d->n_timesteps;
  p->pred = pred; p->x = x; p->xp = x_prev;
  p->prs = d->pred_stride; p->xrs = d->x_stride; p->xprs = d->x_prev_stride;
  p->t = (const long long*)t;
  p->plv = d->posterior_log_variance; p->c1 = d->coef1; p->c2 = d->coef2;
  p->ra = d->sqrt_recip_alphas_cumprod; p->rm = d->sqrt_recipm1_alphas_cumprod;
  p->clamp = d->clip_denoised ? 1 : 0;
  long long free_elems = (long long)H * D;
  for (int k = 0; k < d->n_cond; ++k) {
    const int h = d->cond_index[k];
    if (h < 0 || h >= H) return fail(TREBI_BAD_SHAPE, "conditioned index %d outside the horizon", h);
    bool again = false;                                   // the same index twice covers its elements once
    for (int j = 0; j < k; ++j) again = again || d->cond_index[j] == h;
    if (again) continue;
    p->skip_lo[p->n_skip] = h * D + d->action_dim;
    p->skip_hi[p->n_skip] = h * D + d->action_dim + d->observation_dim;
    ++p->n_skip;
    free_elems -= d->observation_dim;
  }
  p->half_const = 0.5 * (double)free_elems;
  return 0;
}

extern "C" int trebi_transition_logp(trebi_ctx* ctx, const trebi_transition_desc* d, const float* pred, const float* x,
                                     const float* x_prev, const int64_t* t, int64_t B, float* logp, void* stream) {
  TransP p{};
  if (int e = transition_args(ctx, d, pred, x, x_prev, t, B, &p)) return e;
  if (B == 0) return 0;
  if (!logp) return fail(TREBI_BAD_ARG, "logp is null");
  p.logp = logp;
  ON_DEVICE(ctx);
  HIPCHK(launch_transition(p, 0, (hipStream_t)stream));
  return 0;
}

extern "C" int trebi_transition_logp_grad(trebi_ctx* ctx, const trebi_transition_desc* d, const float* pred, const float* x,
                                          const float* x_prev, const int64_t* t, const float* grad_logp, int64_t B, float* grad_pred,
                                          void* stream) {
  TransP p{};
  if (int e = transition_args(ctx, d, pred, x, x_prev, t, B, &p)) return e;
  if (B == 0) return 0;
  if (!grad_logp || !grad_pred) return fail(TREBI_BAD_ARG, "null argument");
  p.g = grad_logp;
  p.dpred = grad_pred;
  ON_DEVICE(ctx);
  HIPCHK(launch_transition(p, 1, (hipStream_t)stream));
  return 0;
}
