// pico_amd/csrc/rope.hip -- rotary positions: the heads of activations turned in pairs by
// their token's position, and the gradient turned back.
#include <math.h>

#include "rope.h"

namespace {

using namespace pk;

constexpr int kThreads = 256;

// Bound by HBM: x is read and y written once, a token's angles are shared by its heads.
// 16384 tokens of 32 heads of 128, 64 turned: 104 us (5.2 TB/s; a large copy 5.1); 8192 of 24
// heads of 64: 20 (5.1); 64 tokens of 12 heads, as a launch and its loads take: 3.2.
template <bool EVEN, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(int64_t N, int T, TurnArgs g, RopeArgs r,
                                                        const int32_t* __restrict__ positions) {
    __shared__ __align__(16) float tc[kTurnTable], ts[kTurnTable];
    const int64_t t0 = (int64_t)blockIdx.x * T;
    turn_rows<EVEN, INTER>(
        g, r, t0, (int)(N - t0 < T ? N - t0 : T), g.H,
        [&](int t, int& pos) {
            pos = positions[t0 + t];
            return true;
        },
        tc, ts);
}

}  // namespace

extern "C" int pk_rope_freqs(int64_t rot, double base, int scaling, double factor, double length,
                             double low, double high, double* freqs) {
    if(rot < 0 || rot % 2 || rot > kTurnHead || (rot > 0 && !freqs))
        return fail("pk_rope_freqs: rot must be even, 0 to %d, and freqs not NULL", kTurnHead);
    if(scaling < PK_ROPE_PLAIN || scaling > PK_ROPE_PARTS)
        return fail("pk_rope_freqs: unknown scaling %d", scaling);
    if(!(base > 0.0) || !isfinite(base) ||
       (scaling != PK_ROPE_PLAIN && (!(factor > 0.0) || !isfinite(factor))))
        return fail("pk_rope_freqs: base and factor must be positive and finite");
    if(scaling == PK_ROPE_PARTS &&
       (!(length > 0.0) || !isfinite(length) || !isfinite(low) || !isfinite(high) || !(low < high)))
        return fail("pk_rope_freqs: scaling by parts needs a length above 0 and low < high");
    if(scaling == PK_ROPE_NTK && rot > 2) base *= pow(factor, (double)rot / (double)(rot - 2));
    for(int64_t i = 0; i < rot / 2; ++i) {
        double f = pow(base, -2.0 * (double)i / (double)rot);
        if(scaling == PK_ROPE_LINEAR) f /= factor;
        if(scaling == PK_ROPE_PARTS) {
            const double turns = length * f / (2.0 * M_PI);
            const double g = fmin(1.0, fmax(0.0, (turns - low) / (high - low)));
            f *= g + (1.0 - g) / factor;
        }
        freqs[i] = f;
    }
    return PK_OK;
}

extern "C" int pk_rope_f32(int64_t N, int64_t H, int64_t hd, const PkRope* rope,
                           const int32_t* positions, const float* x, int64_t ldx, float* y,
                           int64_t ldy, int flags, pk_stream_t stream) {
    if(N < 0 || H < 1 || hd < 1 || hd > kTurnHead || H > (1 << 20) / hd || N > ((int64_t)1 << 24) - 1)
        return fail("pk_rope_f32: N %lld, H %lld, hd %lld: 0 <= N < 2^24, 1 <= hd <= %d, H*hd <= 2^20",
                    (long long)N, (long long)H, (long long)hd, kTurnHead);
    if(!rope || !rope_ok(rope, hd))
        return fail("pk_rope_f32: rope must have an even rot of 0 to hd, and its frequencies");
    if(N == 0) return PK_OK;
    if(!positions || !x || !y) return fail("pk_rope_f32: NULL pointer");
    if(ldx < H * hd || ldy < H * hd)
        return fail("pk_rope_f32: row strides must be at least H*hd = %lld", (long long)(H * hd));
    const RopeArgs r = rope_args(rope);
    TurnArgs g;
    const bool even = turn_args(g, r, H, hd, x, ldx, y, ldy, flags);
    const int T = turn_tokens(N, H, r.half);
    const unsigned grid = (unsigned)((N + T - 1) / T);
    auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, as_stream(stream)>>>(N, T, g, r, positions); };
    if(r.interleaved)
        even ? go(rope_kernel<true, true>) : go(rope_kernel<false, true>);
    else
        even ? go(rope_kernel<true, false>) : go(rope_kernel<false, false>);
    return launch_status("pk_rope_f32");
}
