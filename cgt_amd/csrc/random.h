// Counter-based random numbers for dropout (Philox4x32 of Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011, with 7 rounds: the fewest that paper
// reports as passing BigCrush).  The numbers are a function of (seed, step, channel, group), so
// a mask is formed again wherever it is needed and never stored.
#pragma once
#include "common.h"

namespace cgt_amd {

// rng[0] = seed (the key), rng[1] = step (its low 32 bits count); device memory, read by the
// kernel, so that a captured graph draws new masks when the host changes the step.
struct RngState {
    unsigned k0, k1, step, channel;
};
__device__ __forceinline__ RngState load_rng(const long long* rng, unsigned channel) {
    const unsigned long long seed = (unsigned long long)rng[0];
    RngState s;
    s.k0 = (unsigned)seed;
    s.k1 = (unsigned)(seed >> 32);
    s.step = (unsigned)rng[1];
    s.channel = channel;
    return s;
}

// Eight 16-bit numbers of a group: number e is half e & 1 of word e >> 1.
__device__ __forceinline__ void random_group(const RngState& s, unsigned long long group, unsigned (&w)[4]) {
    unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32), c2 = s.channel, c3 = s.step;
    unsigned k0 = s.k0, k1 = s.k1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}
__device__ __forceinline__ unsigned random16(const unsigned (&w)[4], int e) { return (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu; }

// The probability as the generator's 16-bit numbers resolve it: an element is dropped when its
// number is below `threshold`; `scale` is the reciprocal of the share that is kept, exactly.
struct DropoutRate {
    unsigned threshold;
    float scale;
};
// false (with the message set): p is not in [0, 1) or rounds to 1
inline bool dropout_rate(double p, const char* what, DropoutRate* rate) {
    const double t = p * 65536.0 + 0.5;
    if (!(p >= 0.0 && t < 65536.0)) {
        set_error("%s: the dropout probability must be at least 0 and below 1 by 2^-16 or more (got %g)", what, p);
        return false;
    }
    rate->threshold = (unsigned)t;
    rate->scale = 65536.0f / (float)(65536u - rate->threshold);
    return true;
}

}  // namespace cgt_amd
