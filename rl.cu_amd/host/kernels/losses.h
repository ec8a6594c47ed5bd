// Loss operators for C++ callers: what the reference's trainers launch between forward and backward (log-softmax gather,
// src/model/qwen3.cu:91,170; grpo_loss_kernel, include/training/GRPO_trainer.h:452-517) and a preference loss, forwarding
// to the C ABI of librlx_adamw.so (include/rlx_adamw.h states the formulas).  Like launch_adamw_*, these abort with a message
// if the library reports an error.
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <vector>

#include "kernels/adamw.h"
#include "rlx_adamw.h"

// Scratch memory of the loss operators, grown when a call needs more.  One per stream: calls on one stream may share it,
// calls that can overlap may not.  What was handed out before stays allocated as long as the object, because a recorded graph
// may still use it (sizes at least double, so that is less than the last block once more).  A call that is to be
// recorded has to be made once before, or reserve() called: nothing can be allocated while a stream is recorded.
// A copy starts without memory, and an assignment keeps what it has: there is nothing in it to copy.
class LossWorkspace {
public:
    LossWorkspace() = default;
    LossWorkspace(const LossWorkspace&) {}
    LossWorkspace& operator=(const LossWorkspace&) { return *this; }
    ~LossWorkspace() { for (void* p : blocks_) (void)hipFree(p); }

    void* reserve(int64_t bytes) {
        if (bytes < 0) RLX_CHECK(RLX_ERR_INVALID_ARG);
        if (bytes > bytes_) {
            const int64_t size = bytes > 2 * bytes_ ? bytes : 2 * bytes_;
            void* p = nullptr;
            check(hipMalloc(&p, (size_t)size));
            blocks_.push_back(p);
            bytes_ = size;
        }
        return blocks_.empty() ? nullptr : blocks_.back();
    }
    int64_t bytes() const { return bytes_; }

private:
    static void check(hipError_t e) {
        if (e == hipSuccess) return;
        fprintf(stderr, "loss workspace: %s\n", hipGetErrorString(e));
        exit(1);
    }
    std::vector<void*> blocks_;             // the last one is in use
    int64_t bytes_ = 0;                     // its size
};

// Rows of contiguous logits, or of logits whose rows lie row_stride elements apart.
inline rlx_logits logit_rows(void* data, int dtype, int64_t rows, int64_t vocab, int64_t row_stride = 0) {
    rlx_logits x = {data, rows, vocab, row_stride ? row_stride : vocab, 0, 0, dtype, 0};
    return x;
}

inline void launch_token_logprob(const rlx_logits& x, const int* targets, float temperature, float* logp, float* lse,
                                 float* entropy, LossWorkspace& ws, hipStream_t stream = 0) {
    const int64_t bytes = rlx_token_logprob_workspace(&x);
    void* scratch = ws.reserve(bytes);
    RLX_CHECK(rlx_token_logprob(&x, targets, RLX_INDEX_I32, temperature, logp, lse, entropy, scratch, ws.bytes(),
                                (void*)stream));
}

inline void launch_token_logprob_backward(const rlx_logits& x, const int* targets, float temperature, const float* lse,
                                          const float* entropy, const float* dlogp, const float* dentropy,
                                          const rlx_logits& dx, hipStream_t stream = 0, const float* logp = nullptr) {
    RLX_CHECK(rlx_token_logprob_backward_logp(&x, targets, RLX_INDEX_I32, temperature, lse, entropy, logp, dlogp, dentropy,
                                              &dx, (void*)stream));
}

inline void launch_policy_loss(const float* logp, int64_t tokens, const rlx_policy_args& args, float* dlogp,
                               float* dentropy, rlx_policy_stats* stats, LossWorkspace& ws, hipStream_t stream = 0) {
    void* scratch = ws.reserve(rlx_policy_loss_workspace(tokens, args.n_seqs));
    RLX_CHECK(rlx_policy_loss(logp, tokens, &args, dlogp, dentropy, stats, scratch, ws.bytes(), (void*)stream));
}

inline void launch_policy_loss_logits(const rlx_logits& x, const int* targets, float temperature,
                                      const rlx_policy_args& args, float* logp, float* entropy, const rlx_logits& dx,
                                      rlx_policy_stats* stats, LossWorkspace& ws, hipStream_t stream = 0) {
    void* scratch = ws.reserve(rlx_policy_loss_logits_workspace(&x, args.n_seqs));
    RLX_CHECK(rlx_policy_loss_logits(&x, targets, RLX_INDEX_I32, temperature, &args, logp, entropy, &dx, stats, scratch,
                                     ws.bytes(), (void*)stream));
}

inline void launch_preference_loss(const float* logp, int64_t tokens, const rlx_preference_args& args, float* dlogp,
                                   float* rewards, rlx_preference_stats* stats, LossWorkspace& ws,
                                   hipStream_t stream = 0) {
    void* scratch = ws.reserve(rlx_preference_loss_workspace(tokens, args.n_pairs));
    RLX_CHECK(rlx_preference_loss(logp, tokens, &args, dlogp, rewards, stats, scratch, ws.bytes(), (void*)stream));
}
