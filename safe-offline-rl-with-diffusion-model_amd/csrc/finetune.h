// Kernel arguments and launchers of the fine-tuning operators (gradnorm.hip, policy.inl, policy.hip, pairs.hip, transition.hip), shared with the host side
// (finetune.inl).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace trebi {

// ---- global gradient norm over many tensors ------------------------------------------------------------------
// The set's table lives in device memory: the chunks that the tensors are cut into (a chunk: consecutive elements of one
// tensor).  Workgroup w takes the chunks w, w + n_blocks, ..., so that at any moment the workgroups read and write one
// moving window of memory.
struct GradChunk { void* p; long long out_off; int len; int dtype; };
constexpr int GRAD_BLOCKS = 2048;          // workgroups of 256 threads at most: 8 on each CU
struct GradP {
  const GradChunk* chunks;
  int n_chunks, n_blocks, norm_type;       // 0 two-norm, 1 one-norm, 2 largest magnitude
  int stream_loads, stream_stores;         // past the caches: nothing will read it from there
  int one_each;                            // one chunk of at most 4096 elements for each workgroup
  float grad_scale, max_norm;
  float* out;                              // flat float32 copy, or null: in place
  float* norm_out;                         // [1] or null
  double* part;                            // [n_blocks]
};
hipError_t launch_grad_partials(const GradP& p, hipStream_t st);
hipError_t launch_grad_finish(const GradP& p, float* coef_out, hipStream_t st);     // norm and (coef_out) the factor
hipError_t launch_grad_scale(const GradP& p, hipStream_t st);

// ---- which tokens count ---------------------------------------------------------------------------------------
struct TokenP {
  long long rows, len, n;                  // padded: n = rows * len; packed: n tokens, rows sequences
  int packed;
  const int* lengths;                      // padded: [rows] or null
  const int* cu;                           // packed: [rows + 1]
  const unsigned char* mask;               // or null
  long long mrs, mcs;                      // its row / column strides
};
struct NormPart { long long tokens, rows; };
constexpr int COUNT_BLOCKS = 256;          // partial counts
constexpr int LOSS_PARTS = 1280;          // partial sums the policy loss may leave
constexpr int LOSS_VALS = 5;

struct PolicyP {
  TokenP tk;
  const void *lp, *old, *ref;              // old / ref may be null
  long long lrs, lcs, ors, ocs, rrs, rcs;
  const float* adv;
  long long ars, acs;                      // acs 0: one advantage a row
  void* grad;                              // contiguous, the type of lp; or null
  double hi, lo, dual;                     // borders of the log ratio
  float fhi, flo, fdual;                   // the same, rounded
  float vhi, vlo, vdual;                   // the ratio taken beyond them
  float kl_coef;
  int kl, mode;                            // 1..3; 0 token mean, 1 mean over sequences, 2 a given denominator
  double fixed;                            // mode 2: 1 / denominator; else > 0: 1 / count known on the host, 0: from `np`
  float gscale;
  NormPart* np;
  int nnp;                                 // partial counts written (0: none, the kernel counts the rows itself)
  int* counts;                             // [rows] valid tokens of a row under a mask, or null
  double* part;                            // [LOSS_VALS][LOSS_PARTS]
  double* weight;                          // the weight, from the loss kernel to the one that finishes
  float* stats;                            // [5]
  long long per;                           // tokens of a workgroup
  int early;                               // load tokens before it is known which of them count
  int flat;                                // every view is contiguous and rows are not tiny: vector loads across rows
};
hipError_t launch_token_counts(PolicyP& p, hipStream_t st);     // sets p.nnp
hipError_t launch_policy(const PolicyP& p, int dtype, int blocks, hipStream_t st);
hipError_t launch_policy_finish(const PolicyP& p, int blocks, hipStream_t st);

struct PairP {
  TokenP tk;                               // rows = 2 * pairs: chosen rows first
  long long pairs;
  const void *lp, *ref;                    // ref may be null
  long long lrs, lcs, rrs, rcs;
  const float* weights;                    // [pairs] or null
  void* grad;                              // contiguous, or null
  double beta, margin, inv_p;              // inv_p = 1 / denominator
  float smooth, gscale;
  int kind, average;                       // 0 sigmoid, 1 hinge, 2 ipo
  float *rew_c, *rew_r;                    // [pairs]
  double* part;                            // [nparts][4]: loss, hits, z, pairs that count
  int nparts;                              // workgroups, or pairs where rows are split
  float* stats;                            // [3]
  int group;                               // threads of a pair (whole-pair kernel)
  int splits;                              // workgroups of a row (split kernels)
  double* rowpart;                         // [rows][splits][2]: sum, count
};
hipError_t launch_pairs_whole(const PairP& p, int dtype, hipStream_t st);     // of p.nparts workgroups
hipError_t launch_pairs_split(const PairP& p, int dtype, hipStream_t st);
hipError_t launch_pairs_finish(const PairP& p, hipStream_t st);

struct TransP {
  long long B;
  int H, D, T;
  const float *pred, *x, *xp;
  long long prs, xrs, xprs;                // candidate strides
  const long long* t;
  const float *plv, *c1, *c2, *ra, *rm;    // ra / rm null: the net predicts x0
  int clamp;
  int n_skip, skip_lo[4], skip_hi[4];      // element ranges of a candidate that a condition overwrites
  double half_const;                       // free elements / 2
  float* logp;                             // forward [B]
  const float* g;                          // backward [B]
  float* dpred;                            // backward [B, H, D] contiguous
};
hipError_t launch_transition(const TransP& p, int backward, hipStream_t st);

}  // namespace trebi
