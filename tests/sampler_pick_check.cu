/* Host-side check of the device sampler's walk over probabilities (sm_mult_pick
 * in kc_sampler.cuh), run by tests/test_sampler_pick.py on the CPU: no kernel is
 * launched and no device is needed.
 *
 * stdin: "n barred", then n floats, the probabilities. The stretches' sums are
 * made as the kernel's threads make them. Of the 2^24 coins those within 40 of
 * where the running sum stands after each stretch are tried, the 4096 largest,
 * and every 997th. Prints how many were tried, how many chose a token of
 * probability 0, and how many chose one whose own interval of the cumulative
 * sums (in 64 bits) is further than 2^-14 from the coin (1024 roundings of sums
 * below 1 + 2^-10 or so, 2^-24 at most each). */
#include <cmath>
#include <cstdio>
#include <vector>

#include "kc_sampler.cuh"

using namespace kc;

int main() {
    int n, barred;
    if (std::scanf("%d %d", &n, &barred) != 2) return 1;
    std::vector<float> p(n), csum(SM_THREADS, 0.0f);
    for (float &x : p)
        if (std::scanf("%f", &x) != 1) return 1;
    const int chunk = (n + SM_THREADS - 1) / SM_THREADS;
    std::vector<double> cum(n + 1, 0.0);
    for (int i = 0; i < n; i++) {
        csum[i / chunk] += p[i];
        cum[i + 1] = cum[i] + p[i];
    }
    std::vector<long long> coins;
    float at = 0.0f;
    for (int t = 0; t < SM_THREADS; t++) {
        at += csum[t];
        for (long long d = -40; d <= 40; d++) coins.push_back((long long)(at * 16777216.0f) + d);
    }
    for (long long c = (1 << 24) - 4096; c < 1 << 24; c++) coins.push_back(c);
    for (long long c = 0; c < 1 << 24; c += 997) coins.push_back(c);
    long long tried = 0, zero = 0, far = 0;
    for (long long c : coins) {
        if (c < 0 || c >= 1 << 24) continue;
        const float coin = (float)c / 16777216.0f;
        const int tok = sm_mult_pick(p.data(), csum.data(), SM_THREADS, chunk, n, coin, barred != 0);
        if (tok < 0 || tok >= n) return 1;
        tried++;
        zero += !(p[tok] > 0.0f);
        far += coin < cum[tok] - std::ldexp(1.0, -14) || coin > cum[tok + 1] + std::ldexp(1.0, -14);
    }
    std::printf("%lld %lld %lld\n", tried, zero, far);
    return 0;
}
