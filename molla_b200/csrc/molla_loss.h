// Logprobs of given tokens and the losses over them (molla_loss.cu), called by the entry points in molla_sample.cu.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

// A block of logits and what every one of these calls says about it.
struct LossArgs {
    const void *logits; int type; long long row_stride; int B, V;
    const int *tokens; const float *temperature;
    bool follows;                // the launch is behind another one of the same call
    // outputs of a row (any may be nullptr, but `logprob` and `status` only in a backward pass, which touches them and `loss` where a row's logits did not come in time)
    float *logprob; float *logprob_lo; float *entropy; float *depth; float *stats; unsigned int *status;   // logprob_lo: what the logprob's rounding leaves out; depth: sum p (max - z)
    // the gradient in the logits' type, or nullptr
    void *grad; long long grad_stride;
    // the row's derivatives, where they are given: by logprob (nullptr = the policy loss has them) and by entropy
    const float *g_logprob; const float *g_entropy; const float *in_stats; const float *in_entropy; const float *in_depth;   // (one of the last two)
    // the policy loss
    const float *old_logprob; const float *advantage; const float *weight; const float *ref_logprob;
    float clip_low, clip_high, kl_coef, entropy_coef, scale, grad_scale;
    float *loss; float *row_loss; float *kl; unsigned char *clipped;
#ifdef MOLLA_SAMPLE_TESTING
    int knobs;                   // experiment switches (0 = production behaviour)
#endif
};

// The preference loss between its two passes over the logits.
struct PairArgs {
    int B, n_pairs;
    const int *tokens; const int *off; const float *logprob; const float *logprob_lo; const float *ref_logprob; const float *weight; const unsigned int *row_status;
    float beta, smoothing, scale, grad_scale;
    float *loss; float *pair_loss; float *margin; float *seq_logratio; unsigned int *pair_status;
    float *g_logprob;            // [B] the rows' derivatives, or nullptr
};

cudaError_t molla_loss_score(const LossArgs &a, cudaStream_t st);      // logprobs, entropies, stats
cudaError_t molla_loss_backward(const LossArgs &a, cudaStream_t st);   // the gradient from stats and the rows' derivatives
cudaError_t molla_loss_policy(const LossArgs &a, cudaStream_t st);     // the policy loss and its gradient
cudaError_t molla_loss_pairs(const PairArgs &a, cudaStream_t st);
