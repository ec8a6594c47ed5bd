// test_losses_host.cpp
//
// The loss operators from C++ on a GPU, each against an inline loop in double on the host:
//   1. log-probabilities, entropies and their gradient         2. policy loss from log-probabilities
//   3. policy loss from logits, the gradient over the logits    4. preference loss
//   5. OptimStep::policy_step: the logits are the parameters themselves (one row of weights per token), so the
//      gradient in the pool, the norm and the update can be checked end to end (the update against the C oracle, bit for bit)
//   6. a recorded call replayed after its LossWorkspace has grown
// Bounds: FP32 arithmetic on values of size 1 to 10 over 101 logits: 1e-5 is more than ten times what its roundings add up to
// (each of at most 6e-8 of the value, fewer than ten of them on the way to a result, plus sums of 101 positive terms).
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <type_traits>
#include <vector>

#include "training/optim_step.h"

extern "C" {
void orc_adamw_fp32(float*, const float*, float*, float*, int64_t, float, float, float, float, float, float, float);
}

static int g_fails = 0;
#define PASS(name) printf("[PASS] %s\n", (name))
#define FAIL(name, ...) do { printf("[FAIL] %s: ", (name)); printf(__VA_ARGS__); printf("\n"); g_fails++; } while (0)

template <typename T>
struct Dev {
    T* p = nullptr;
    size_t n;
    explicit Dev(const std::vector<T>& h) : n(h.size()) {
        HIP_CHECK(hipMalloc((void**)&p, n * sizeof(T) + 64));
        HIP_CHECK(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    explicit Dev(size_t count) : Dev(std::vector<T>(count)) {}
    ~Dev() { (void)hipFree(p); }
    std::vector<T> get() const {
        std::vector<T> h(n);
        HIP_CHECK(hipDeviceSynchronize());
        HIP_CHECK(hipMemcpy(h.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return h;
    }
};

static uint32_t g_seed = 12345;
static float rnd(float lo, float hi) {
    g_seed = g_seed * 1664525u + 1013904223u;
    return lo + (hi - lo) * (float)(g_seed >> 8) / 16777216.0f;
}
static std::vector<float> randoms(size_t n, float lo, float hi) {
    std::vector<float> v(n);
    for (float& x : v) x = rnd(lo, hi);
    return v;
}

static const int ROWS = 14, VOCAB = 101, SEQS = 3;
static const std::vector<int> CU = {1, 5, 5, 13};              // token 0 and the last belong to no sequence

struct Batch {
    std::vector<float> logits = randoms((size_t)ROWS * VOCAB, -4.0f, 4.0f), old, ref, adv = randoms(SEQS, -1.0f, 1.0f);
    std::vector<int> targets;
    std::vector<uint8_t> mask;
    std::vector<double> logp, lse, ent;
    Batch() {
        for (int r = 0; r < ROWS; r++) {
            targets.push_back((int)rnd(0.0f, (float)VOCAB - 0.01f));
            mask.push_back(r % 5 != 2);
            double sum = 0.0, h = 0.0;
            for (int j = 0; j < VOCAB; j++) sum += exp((double)at(r, j));
            lse.push_back(log(sum));
            for (int j = 0; j < VOCAB; j++) h -= exp((double)at(r, j)) / sum * ((double)at(r, j) - lse[(size_t)r]);
            ent.push_back(h);
            logp.push_back((double)at(r, targets[(size_t)r]) - lse[(size_t)r]);
            old.push_back((float)logp[(size_t)r] - rnd(-0.15f, 0.15f));       // inside the clip of 0.2
            ref.push_back((float)logp[(size_t)r] + rnd(-0.5f, 0.5f));
        }
    }
    float at(int r, int j) const { return logits[(size_t)r * VOCAB + j]; }
    int seq(int r) const {
        for (int s = 0; s < SEQS; s++) if (r >= CU[(size_t)s] && r < CU[(size_t)s + 1]) return mask[(size_t)r] ? s : -1;
        return -1;
    }
    // weight, gradient of the log-probability and loss of a token (mean over sequences of means)
    double weight(int r) const {
        int n = 0;
        for (int q = 0; q < ROWS; q++) n += seq(q) >= 0 && seq(q) == seq(r);
        return seq(r) < 0 ? 0.0 : 1.0 / (SEQS * (double)n);
    }
    double slope(int r, double kl) const {
        if (seq(r) < 0) return 0.0;
        return weight(r) * (-(double)adv[(size_t)seq(r)] * exp(logp[(size_t)r] - old[(size_t)r]) -
                            kl * expm1((double)ref[(size_t)r] - logp[(size_t)r]));
    }
    double loss(double kl) const {
        double l = 0.0;
        for (int r = 0; r < ROWS; r++) {
            if (seq(r) < 0) continue;
            const double d = (double)ref[(size_t)r] - logp[(size_t)r];
            l += weight(r) * (-(double)adv[(size_t)seq(r)] * exp(logp[(size_t)r] - old[(size_t)r]) + kl * (expm1(d) - d));
        }
        return l;
    }
    double dlogit(int r, int j, double g) const {
        return g * ((j == targets[(size_t)r]) - exp((double)at(r, j) - lse[(size_t)r]));
    }
};

static rlx_policy_args policy_args(const Dev<float>& old, const Dev<float>& ref, const Dev<float>& adv, const Dev<uint8_t>& mask,
                                   const Dev<int>& cu, float kl) {
    rlx_policy_args a;
    memset(&a, 0, sizeof(a));
    a.old_logp = old.p; a.ref_logp = ref.p; a.advantages = adv.p; a.mask = mask.p; a.cu_seqlens = cu.p; a.n_seqs = SEQS;
    a.clip_low = 0.2f; a.clip_high = 0.2f; a.kl_coef = kl; a.norm = 1.0f; a.grad_scale = 1.0f;
    a.reduction = RLX_LOSS_SEQUENCE_MEAN;
    return a;
}

static void test_logprob() {
    const char* name = "token log-probabilities and their gradient";
    Batch b;
    Dev<float> x(b.logits), logp(ROWS), lse(ROWS), ent(ROWS), dx((size_t)ROWS * VOCAB);
    Dev<int> t(b.targets);
    const std::vector<float> g = randoms(ROWS, -1.0f, 1.0f);
    Dev<float> dlogp(g);
    LossWorkspace ws;
    const rlx_logits rows = logit_rows(x.p, RLX_DTYPE_F32, ROWS, VOCAB), out = logit_rows(dx.p, RLX_DTYPE_F32, ROWS, VOCAB);
    launch_token_logprob(rows, t.p, 1.0f, logp.p, lse.p, ent.p, ws);
    launch_token_logprob_backward(rows, t.p, 1.0f, lse.p, nullptr, dlogp.p, nullptr, out);
    const auto hl = logp.get(), he = ent.get(), hs = lse.get(), hd = dx.get();
    double worst = 0.0;
    for (int r = 0; r < ROWS; r++) {
        worst = fmax(worst, fmax(fabs(hl[r] - b.logp[r]), fmax(fabs(he[r] - b.ent[r]), fabs(hs[r] - b.lse[r]))));
        for (int j = 0; j < VOCAB; j++) worst = fmax(worst, fabs(hd[(size_t)r * VOCAB + j] - b.dlogit(r, j, g[(size_t)r])));
    }
    if (worst < 1e-5) PASS(name); else FAIL(name, "off by %g", worst);
}

static void test_policy() {
    const char* name = "policy loss from log-probabilities";
    Batch b;
    std::vector<float> lp(b.logp.begin(), b.logp.end());
    Dev<float> logp(lp), old(b.old), ref(b.ref), adv(b.adv), dlogp(ROWS);
    Dev<uint8_t> mask(b.mask);
    Dev<int> cu(CU);
    Dev<rlx_policy_stats> stats(1);
    LossWorkspace ws;
    launch_policy_loss(logp.p, ROWS, policy_args(old, ref, adv, mask, cu, 0.1f), dlogp.p, nullptr, stats.p, ws);
    const auto g = dlogp.get();
    const rlx_policy_stats s = stats.get()[0];
    double worst = fabs(s.loss - b.loss(0.1));
    int n = 0;
    for (int r = 0; r < ROWS; r++) { worst = fmax(worst, fabs(g[r] - b.slope(r, 0.1))); n += b.seq(r) >= 0; }
    if (worst < 1e-5 && s.tokens == n && s.clip_fraction == 0.0f) PASS(name); else FAIL(name, "off by %g, %lld tokens", worst, (long long)s.tokens);
}

static void test_policy_logits() {
    const char* name = "policy loss from logits, gradient over the logits";
    Batch b;
    Dev<float> x(b.logits), logp(ROWS), old(b.old), ref(b.ref), adv(b.adv);
    Dev<int> t(b.targets), cu(CU);
    Dev<uint8_t> mask(b.mask);
    Dev<rlx_policy_stats> stats(1);
    LossWorkspace ws;
    const rlx_logits rows = logit_rows(x.p, RLX_DTYPE_F32, ROWS, VOCAB);
    launch_policy_loss_logits(rows, t.p, 1.0f, policy_args(old, ref, adv, mask, cu, 0.1f), logp.p, nullptr, rows, stats.p, ws);
    const auto g = x.get(), lp = logp.get();
    double worst = fabs(stats.get()[0].loss - b.loss(0.1));
    for (int r = 0; r < ROWS; r++) {
        worst = fmax(worst, fabs(lp[r] - (b.seq(r) >= 0 ? b.logp[r] : 0.0)));
        for (int j = 0; j < VOCAB; j++) worst = fmax(worst, fabs(g[(size_t)r * VOCAB + j] - b.dlogit(r, j, b.slope(r, 0.1))));
    }
    if (worst < 1e-5) PASS(name); else FAIL(name, "off by %g", worst);
}

static void test_preference() {
    const char* name = "preference loss";
    const std::vector<float> lp = randoms(11, -3.0f, 0.0f), rf = randoms(11, -3.0f, 0.0f);
    const std::vector<int> cu = {0, 3, 4, 9, 11};                 // chosen: [0,3) [3,4), rejected: [4,9) [9,11)
    Dev<float> logp(lp), ref(rf), dlogp(11), rewards(4);
    Dev<int> offsets(cu);
    Dev<rlx_preference_stats> stats(1);
    rlx_preference_args a;
    memset(&a, 0, sizeof(a));
    a.ref_logp = ref.p; a.cu_seqlens = offsets.p; a.n_pairs = 2; a.beta = 0.5f; a.grad_scale = 1.0f;
    LossWorkspace ws;
    launch_preference_loss(logp.p, 11, a, dlogp.p, rewards.p, stats.p, ws);
    double r[4] = {0, 0, 0, 0}, loss = 0.0, worst = 0.0;
    for (int s = 0; s < 4; s++) for (int t = cu[(size_t)s]; t < cu[(size_t)s + 1]; t++) r[s] += 0.5 * ((double)lp[(size_t)t] - rf[(size_t)t]);
    const auto g = dlogp.get(), hr = rewards.get();
    for (int p = 0; p < 2; p++) {
        const double x = r[p] - r[p + 2], slope = -0.5 / (1.0 + exp(x)) / 2.0;
        loss += log1p(exp(-x)) / 2.0;
        for (int side = 0; side < 2; side++)
            for (int t = cu[(size_t)(p + 2 * side)]; t < cu[(size_t)(p + 2 * side) + 1]; t++)
                worst = fmax(worst, fabs(g[(size_t)t] - (side ? -slope : slope)));
    }
    for (int s = 0; s < 4; s++) worst = fmax(worst, fabs(hr[(size_t)s] - r[s]));
    worst = fmax(worst, fabs(stats.get()[0].loss - loss));
    if (worst < 1e-5) PASS(name); else FAIL(name, "off by %g", worst);
}

// Two micro-batches over the same rows of weights: the pool's gradient is the mean of the two.
static void test_policy_step() {
    const char* name = "policy_step: loss, gradients, norm and update";
    Batch b;
    const size_t n32 = (size_t)ROWS * VOCAB, n16 = 512;
    ParamPools pools;
    Dev<float> w(b.logits);
    Dev<uint16_t> w16(std::vector<uint16_t>(n16, 0x3c00));
    pools.fp16_pool = (half*)w16.p; pools.fp16_pool_elems = n16; pools.proj_elems = n16;
    pools.fp32_pool = w.p; pools.fp32_pool_elems = n32;
    GradPools grads = grad_pools_alloc(pools, 0);
    AdamWOptimizer opt(pools, 1e-2f, 0.9f, 0.999f, 1e-8f, 0.0f);
    OptimStepConfig cfg;
    cfg.max_grad_norm = 1e30f;                                   // measured, not clipped
    OptimStep step(&opt, cfg);
    Dev<float> x(n32), logp(ROWS), old(b.old), ref(b.ref), adv(b.adv);
    Dev<int> t(b.targets), cu(CU);
    Dev<uint8_t> mask(b.mask);
    std::vector<float> host_grad(n32, 0.0f);
    const float kls[2] = {0.1f, 0.3f};
    auto forward = [&](int k) {
        HIP_CHECK(hipMemcpy(x.p, w.p, n32 * 4, hipMemcpyDeviceToDevice));
        OptimStep::PolicyBatch pb;
        pb.logits = logit_rows(x.p, RLX_DTYPE_F32, ROWS, VOCAB);
        pb.targets = t.p;
        pb.args = policy_args(old, ref, adv, mask, cu, kls[k]);
        pb.logp = logp.p;
        return pb;
    };
    auto backward = [&](int, const rlx_logits& d) {                // adds on the host: d loss / d weights is d itself
        std::vector<float> h(n32);
        HIP_CHECK(hipDeviceSynchronize());
        HIP_CHECK(hipMemcpy(h.data(), d.data, n32 * 4, hipMemcpyDeviceToHost));
        for (size_t i = 0; i < n32; i++) host_grad[i] += h[i];
        HIP_CHECK(hipMemcpy(grads.float_pool, host_grad.data(), n32 * 4, hipMemcpyHostToDevice));
    };
    const float loss = step.policy_step(&grads, 2, forward, backward);
    double worst = fabs(loss - (b.loss(0.1) + b.loss(0.3)) / 2.0), sq = 0.0;
    for (int r = 0; r < ROWS; r++)
        for (int j = 0; j < VOCAB; j++) {
            const double want = b.dlogit(r, j, (b.slope(r, 0.1) + b.slope(r, 0.3)) / 2.0);
            worst = fmax(worst, fabs(host_grad[(size_t)r * VOCAB + j] - want));
            sq += want * want;
        }
    worst = fmax(worst, fabs(step.last_grad_norm() - sqrt(sq)));
    std::vector<float> ew = b.logits, m(n32, 0.0f), v(n32, 0.0f);
    orc_adamw_fp32(ew.data(), host_grad.data(), m.data(), v.data(), (int64_t)n32, 1e-2f, 0.9f, 0.999f, 1e-8f, 0.0f,
                   1.0f - powf(0.9f, 1.0f), 1.0f - powf(0.999f, 1.0f));
    const auto got = w.get();
    size_t diff = 0;
    for (size_t i = 0; i < n32; i++) diff += memcmp(&got[i], &ew[i], 4) != 0;
    const bool counted = step.statistics().size() == 2 && step.statistics()[0].tokens == step.statistics()[1].tokens;
    if (worst < 1e-5 && diff == 0 && counted && opt.get_step() == 1) PASS(name);
    else FAIL(name, "off by %g, %zu weights differ, step %d", worst, diff, opt.get_step());
    grad_pools_free(&grads);
}

static_assert(std::is_copy_constructible<OptimStep>::value && std::is_copy_assignable<OptimStep>::value,
              "steps are held by value");

// Rows of equal logits, long enough to need scratch memory: every log-probability is -log(vocabulary).
static void test_workspace_grows() {
    const char* name = "a recorded call replayed after its workspace has grown";
    const int rows = 3, vocab = 20000;
    Dev<float> x((size_t)rows * vocab), logp(rows), lse(rows);
    Dev<int> t(rows);
    const rlx_logits view = logit_rows(x.p, RLX_DTYPE_F32, rows, vocab);
    const int64_t need = rlx_token_logprob_workspace(&view);
    LossWorkspace ws;
    hipStream_t s;
    hipGraph_t graph;
    hipGraphExec_t exec;
    HIP_CHECK(hipStreamCreate(&s));
    launch_token_logprob(view, t.p, 1.0f, logp.p, lse.p, nullptr, ws, s);
    HIP_CHECK(hipStreamSynchronize(s));
    HIP_CHECK(hipStreamBeginCapture(s, hipStreamCaptureModeThreadLocal));
    launch_token_logprob(view, t.p, 1.0f, logp.p, lse.p, nullptr, ws, s);
    HIP_CHECK(hipStreamEndCapture(s, &graph));
    HIP_CHECK(hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0));
    const void* before = ws.reserve(need);
    const bool moved = ws.reserve(need + 1) != before && ws.bytes() >= 2 * need && ws.reserve(need) != before;
    LossWorkspace copy(ws);
    double worst = need > 0 && moved && copy.bytes() == 0 ? 0.0 : 1.0;
    for (int i = 0; i < 3; i++) {
        HIP_CHECK(hipMemcpy(logp.p, std::vector<float>(rows, 7.0f).data(), rows * sizeof(float), hipMemcpyHostToDevice));
        HIP_CHECK(hipGraphLaunch(exec, s));
        HIP_CHECK(hipStreamSynchronize(s));
        for (float v : logp.get()) worst = fmax(worst, fabs(v + log((double)vocab)));
    }
    // 20,000 equal terms of 1 and a logarithm near 10: sums that are exact, and two roundings of 6e-7
    if (worst < 1e-5) PASS(name); else FAIL(name, "off by %g (%lld bytes)", worst, (long long)need);
    (void)hipGraphExecDestroy(exec);
    (void)hipGraphDestroy(graph);
    (void)hipStreamDestroy(s);
}

int main() {
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
        printf("no GPU: this test needs one\n");
        return 2;
    }
    test_logprob();
    test_policy();
    test_policy_logits();
    test_preference();
    test_policy_step();
    test_workspace_grows();
    printf("=== %s (%d failures) ===\n", g_fails ? "FAILED" : "ALL PASSED", g_fails);
    return g_fails;
}
