// The operators of a training step on the `HIP` device (needs an MI355X): group norm, 8-bit checkpoints,
// log-probabilities and the policy loss through the C++ calls, eager and recorded by `Lazy`.
#include <cstdint>

#include "check.hpp"
#include "custos/custos.hpp"

using namespace custos;

namespace {

// Bounds: every value is f32 arithmetic with fewer than 256 roundings on its path, so it is off by at most
// 256 * 2^-24 times the magnitude of its terms, and is rounded once (f32 here: 2^-24 of it, within that).
const double kStep = 256.0 / (1 << 24);

std::vector<float> values(size_t n, uint32_t seed, float scale = 1.0f) {
    std::vector<float> v(n);
    uint32_t s = seed * 2654435761u + 1;
    for (float& x : v) {
        s = s * 1664525u + 1013904223u;
        x = scale * (static_cast<float>(s >> 8) / 8388608.0f - 1.0f);
    }
    return v;
}

void check_close(const char* what, const std::vector<float>& got, const std::vector<double>& want, double scale) {
    if (got.size() != want.size()) return check::fail(__FILE__, __LINE__, std::string(what) + ": length");
    for (size_t i = 0; i < got.size(); i++)
        if (!(std::fabs(got[i] - want[i]) <= kStep * scale))
            return check::fail(__FILE__, __LINE__, std::string(what) + " at " + std::to_string(i) + ": " +
                                                       std::to_string(got[i]) + " for " + std::to_string(want[i]));
}

struct NormRef {
    std::vector<double> out, stats, x_grad, gamma_grad, beta_grad;
};

// relu(h * gamma + beta), its gradients for the out gradient `g`
NormRef norm_ref(const std::vector<double>& x, const std::vector<float>& gamma, const std::vector<float>& beta,
                 const std::vector<float>& g, const GroupNorm& n) {
    NormRef r;
    const size_t per = n.channels / n.groups;
    r.out.resize(x.size()), r.x_grad.resize(x.size());
    r.stats.resize(n.samples * n.groups * 2);
    r.gamma_grad.resize(n.channels), r.beta_grad.resize(n.channels);
    const double count = static_cast<double>(n.positions * per);
    for (size_t s = 0; s < n.samples; s++)
        for (size_t q = 0; q < n.groups; q++) {
            auto at = [&](size_t p, size_t c) { return (s * n.positions + p) * n.channels + q * per + c; };
            double mean = 0, var = 0, g1 = 0, g2 = 0;
            for (size_t p = 0; p < n.positions; p++)
                for (size_t c = 0; c < per; c++) mean += x[at(p, c)] / count;
            for (size_t p = 0; p < n.positions; p++)
                for (size_t c = 0; c < per; c++) var += (x[at(p, c)] - mean) * (x[at(p, c)] - mean) / count;
            const double rstd = 1 / std::sqrt(var + n.eps);
            r.stats[(s * n.groups + q) * 2] = mean, r.stats[(s * n.groups + q) * 2 + 1] = rstd;
            auto slope = [&](size_t p, size_t c) { return r.out[at(p, c)] > 0 ? static_cast<double>(g[at(p, c)]) : 0.0; };
            for (size_t p = 0; p < n.positions; p++)
                for (size_t c = 0; c < per; c++) {
                    const size_t ch = q * per + c;
                    const double h = (x[at(p, c)] - mean) * rstd, z = h * gamma[ch] + beta[ch];
                    r.out[at(p, c)] = z > 0 ? z : 0;
                    r.gamma_grad[ch] += slope(p, c) * h, r.beta_grad[ch] += slope(p, c);
                    g1 += slope(p, c) * gamma[ch] / count, g2 += slope(p, c) * gamma[ch] * h / count;
                }
            for (size_t p = 0; p < n.positions; p++)
                for (size_t c = 0; c < per; c++) {
                    const double h = (x[at(p, c)] - mean) * rstd;
                    r.x_grad[at(p, c)] = rstd * (slope(p, c) * gamma[q * per + c] - g1 - h * g2);
                }
        }
    return r;
}

std::vector<double> wide(const std::vector<float>& v) { return std::vector<double>(v.begin(), v.end()); }

}  // namespace

TEST_CASE(op_group_norm_and_checkpoint) {
    using D = HIP<Base>;
    D device;
    const GroupNorm n{3, 37, 24, 4, CUSTOS_HIP_ACT_RELU, 1e-5};
    const size_t len = n.samples * n.positions * n.channels;
    const std::vector<float> xs = values(len, 1, 2.0f), gs = values(len, 2), gam = values(n.channels, 3), bet = values(n.channels, 4);
    auto x = device.buffer(xs), g = device.buffer(gs), gamma = device.buffer(gam), beta = device.buffer(bet);
    Buffer<float, D> out(device, len), stats(device, n.samples * n.groups * 2), xg(device, len), gg(device, n.channels),
        bg(device, n.channels), scales(device, (len + 127) / 128);
    Buffer<int8_t, D> codes(device, len);

    device.group_norm_impl(x, &gamma, &beta, out, stats, n);
    const NormRef ref = norm_ref(wide(xs), gam, bet, gs, n);
    check_close("out", out.read(), ref.out, 8);
    check_close("stats", stats.read(), ref.stats, 2);
    device.add_group_norm_grad_impl(x, stats, &gamma, &beta, g, &xg, &gg, &bg, n);
    // sums over samples * positions = 111 terms of at most 1, of at most 2 with h
    check_close("x_grad", xg.read(), ref.x_grad, 8);
    check_close("gamma_grad", gg.read(), ref.gamma_grad, 222);
    check_close("beta_grad", bg.read(), ref.beta_grad, 111);
    // a second one is added to it
    device.add_group_norm_grad_impl(x, stats, &gamma, &beta, g, &xg, &gg, &bg, n);
    std::vector<double> twice = ref.x_grad;
    for (double& v : twice) v *= 2;
    check_close("x_grad twice", xg.read(), twice, 16);

    // the checkpoint holds x to within half a scale, and the gradient taken from it is the gradient at what it holds
    device.checkpoint8_impl(x, codes, scales);
    auto held = x.empty_like();
    device.restore8_impl(codes, scales, held, [](auto v) { return v; });
    const std::vector<float> hs = held.read(), sc = scales.read();
    for (size_t i = 0; i < len; i++) CHECK(std::fabs(hs[i] - xs[i]) <= 0.50001f * sc[i / 128]);
    auto from8 = x.empty_like(), from_values = x.empty_like();
    device.add_group_norm_grad8_impl(codes, scales, stats, &gamma, &beta, g, &from8, static_cast<Buffer<float, D>*>(nullptr),
                                     static_cast<Buffer<float, D>*>(nullptr), n, true);
    device.add_group_norm_grad_impl(held, stats, &gamma, &beta, g, &from_values, static_cast<Buffer<float, D>*>(nullptr),
                                    static_cast<Buffer<float, D>*>(nullptr), n, true);
    check_close("x_grad of the checkpoint", from8.read(), wide(from_values.read()), 8);

    // no parameters: ones and zeros
    device.group_norm_impl(x, static_cast<Buffer<float, D>*>(nullptr), static_cast<Buffer<float, D>*>(nullptr), out, stats, n);
    check_close("out without parameters", out.read(),
                norm_ref(wide(xs), std::vector<float>(n.channels, 1), std::vector<float>(n.channels, 0), gs, n).out, 8);

    // lengths that do not fit the sizes
    Buffer<float, D> small(device, len - 1);
    CHECK_THROWS_KIND(device.group_norm_impl(x, &gamma, &beta, small, stats, n), DeviceError::ShapeLengthMismatch);
    CHECK_THROWS_KIND(device.checkpoint8_impl(small, codes, scales), DeviceError::ShapeLengthMismatch);
    CHECK_THROWS_KIND(device.group_norm_impl(x, &gamma, &beta, out, stats, GroupNorm{3, 37, 24, 5}), DeviceError::ShapeLengthMismatch);
    CHECK_THROWS_KIND(device.group_norm_impl(x, &gamma, &beta, out, x, GroupNorm{3, 37, 24, 444}), DeviceError::Backend);
}

TEST_CASE(op_unary_through_a_checkpoint) {
    using D = HIP<Base>;
    D device;
    const size_t len = 1000;
    const std::vector<float> xs = values(len, 5, 3.0f), gs = values(len, 6);
    auto x = device.buffer(xs), g = device.buffer(gs);
    Buffer<float, D> out(device, len), scales(device, 8), held(device, len), grad(device, len);
    Buffer<int8_t, D> codes(device, len);
    device.apply_fn_checkpoint8_impl(x, out, codes, scales, [](auto v) { return v.tanh(); });
    device.restore8_impl(codes, scales, held, [](auto v) { return v; });
    device.add_unary_grad8_impl(codes, scales, grad, g, [](auto v) { return v.tanh().pow(2).neg().add(1); });
    const std::vector<float> hs = held.read();
    std::vector<double> want_out(len), want_grad(len);
    for (size_t i = 0; i < len; i++) {
        want_out[i] = std::tanh(static_cast<double>(xs[i]));
        want_grad[i] = gs[i] * (1 - std::pow(std::tanh(static_cast<double>(hs[i])), 2));
    }
    check_close("tanh", out.read(), want_out, 1);
    check_close("its gradient", grad.read(), want_grad, 1);
    Buffer<float, D> few(device, 7);
    CHECK_THROWS_KIND(device.checkpoint8_impl(x, codes, few), DeviceError::ShapeLengthMismatch);
}

TEST_CASE(op_policy_loss) {
    using D = HIP<Base>;
    D device;
    const size_t rows = 6, vocab = 131;
    const std::vector<float> zs = values(rows * vocab, 7, 4.0f), old = values(rows, 8, 0.25f), ref = values(rows, 9, 0.25f),
                             adv = values(rows, 10, 2.0f), w = {0.25f, 0.25f, 0.0f, 0.25f, 0.5f, 0.25f};
    const std::vector<int32_t> chosen = {0, 130, 5, -1, 64, 7};
    auto z = device.buffer(zs);
    auto labels = device.buffer(chosen);
    Buffer<float, D> logp(device, rows), lse(device, rows), grad(device, rows * vocab), totals(device, 4);
    device.token_logprob_impl(z, labels, logp, &lse, 0.5);
    std::vector<double> want_lse(rows), want_logp(rows);
    for (size_t r = 0; r < rows; r++) {
        double sum = 0;
        for (size_t c = 0; c < vocab; c++) sum += std::exp(zs[r * vocab + c] / 0.5);
        want_lse[r] = std::log(sum);
        want_logp[r] = chosen[r] < 0 ? 0 : zs[r * vocab + chosen[r]] / 0.5 - want_lse[r];
    }
    check_close("lse", lse.read(), want_lse, 16);
    check_close("logp", logp.read(), want_logp, 16);

    // old and reference values near the ones of the policy, so that some rows are clipped and some are not
    std::vector<float> old_logp(rows), ref_logp(rows);
    for (size_t r = 0; r < rows; r++) {
        old_logp[r] = static_cast<float>(want_logp[r]) + old[r];
        ref_logp[r] = static_cast<float>(want_logp[r]) + ref[r];
    }
    PolicyLoss loss;
    loss.clip_low = 0.05, loss.clip_high = 0.1, loss.kl_coef = 0.3, loss.temperature = 0.5;
    auto old_buf = device.buffer(old_logp), ref_buf = device.buffer(ref_logp), adv_buf = device.buffer(adv), w_buf = device.buffer(w);
    device.policy_loss_impl(z, labels, old_buf, &ref_buf, adv_buf, w_buf, &grad, &logp, &totals, loss);
    std::vector<double> want_grad(rows * vocab, 0.0);
    double want_loss = 0;
    for (size_t r = 0; r < rows; r++) {
        if (chosen[r] < 0 || w[r] == 0) continue;
        const double ratio = std::exp(want_logp[r] - old_logp[r]), d = ref_logp[r] - want_logp[r];
        const double clipped = std::min(std::max(ratio, 0.95), 1.1);
        const bool free = ratio * adv[r] <= clipped * adv[r];
        want_loss += w[r] * (0.3 * (std::exp(d) - 1 - d) - std::min(ratio * adv[r], clipped * adv[r]));
        const double by_logp = w[r] * (0.3 * (1 - std::exp(d)) - (free ? ratio * adv[r] : 0.0));
        for (size_t c = 0; c < vocab; c++)
            want_grad[r * vocab + c] = by_logp * ((static_cast<int32_t>(c) == chosen[r] ? 1 : 0) -
                                                  std::exp(zs[r * vocab + c] / 0.5 - want_lse[r])) / 0.5;
    }
    // logp and lse, of at most 16, are off by 16 steps; the loss and the gradient change by at most 4 times that: weights of
    // at most 0.5, ratios of at most 1.3 times advantages of at most 2 (and 0.3 * 1.3), over a temperature of 0.5
    check_close("loss", {totals.read()[0]}, {want_loss}, 64);
    check_close("logits_grad", grad.read(), want_grad, 64);

    // in place of the logits, without the rest
    device.policy_loss_impl(z, labels, old_buf, &ref_buf, adv_buf, w_buf, &z, static_cast<Buffer<float, D>*>(nullptr),
                            static_cast<Buffer<float, D>*>(nullptr), loss);
    CHECK_VEC_EQ(z.read(), grad.read());
    Buffer<float, D> five(device, 5);
    CHECK_THROWS_KIND(device.policy_loss_impl(z, labels, old_buf, &ref_buf, five, w_buf, &grad, &logp, &totals, loss),
                      DeviceError::ShapeLengthMismatch);
}

// a lazy program records the operators like its other launches: one graph, replayed with rewritten inputs
TEST_CASE(op_lazy_run_replays_operators) {
    using D = HIP<Lazy<Base, float>>;
    D device;
    const GroupNorm n{2, 19, 16, 2, CUSTOS_HIP_ACT_RELU, 1e-5};
    const size_t len = n.samples * n.positions * n.channels;
    const std::vector<float> gam = values(n.channels, 11), bet = values(n.channels, 12);
    auto x = device.buffer(values(len, 13));
    auto gamma = device.buffer(gam), beta = device.buffer(bet);
    Buffer<float, D> stats(device, n.samples * n.groups * 2), out(device, len), doubled(device, len);
    device.add_op(std::tie(x, gamma, beta, out, stats),
                  [n](Buffer<float, D>& a, Buffer<float, D>& ga, Buffer<float, D>& be, Buffer<float, D>& o, Buffer<float, D>& st, D& d) {
                      d.group_norm_impl(a, &ga, &be, o, st, n);
                  });
    device.add_op(std::tie(out, doubled), [](Buffer<float, D>& o, Buffer<float, D>& t, D& d) {
        d.apply_fn_impl(o, t, [](auto v) { return v.mul(2); });
    });
    for (uint32_t run = 0; run < 4; run++) {
        const std::vector<float> xs = values(len, 20 + run, 1.0f + run);
        x.write(xs);
        device.run();
        std::vector<double> want = norm_ref(wide(xs), gam, bet, std::vector<float>(len), n).out;
        check_close("out", out.read(), want, 8);
        for (double& v : want) v *= 2;
        check_close("doubled", doubled.read(), want, 16);
    }
    CHECK_EQ(device.graph_builds(), uint64_t(1));
}

int main(int argc, char** argv) { return check::run(argc, argv); }
