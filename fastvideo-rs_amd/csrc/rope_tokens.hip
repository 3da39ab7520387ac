// Rotary positions without tables (declarations: include/fv_sdpa_hip.h): pair (a, b) of token t becomes amplitude * (a c - b s, a s + b c) with
// c, s = cos, sin of 2 pi times the turns position * freq, or, turned back, (a c + b s, b c - a s).
//
// freq counts turns a position in units of 2^-64, so that position * freq modulo 2^64 is the angle's fraction of a turn, exact in
// integers but for freq's own rounding: 2^31 positions are 2^-33 turns off at most, where f32 (or a product in f32) loses the angle at some
// ten thousand. Its nearest quarter turn is taken off and the rest, at most 1/8 turn, goes in f32 (converted, times 2 pi as a float: 2^-26 turns off at most) through the
// series of sin and cos, whose next terms are below 2^-29 and 2^-33. Memory is the bound: a thread makes the angles of its channels once and turns them in all heads. Measured:
// 56637 tokens, 40 + 8 heads of 128 in bf16, half of each turned, out of a fused projection, 274 us, 5.1 TB/s; 65520 tokens, 12 + 12 heads in f32,
// three position axes, 309 us, 5.2 TB/s (a copy of 2 GiB goes at 4.9); 32 tokens 4.7 us.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "../../include/fv_sdpa_hip.h"
#include "fv_common.h"
#include "fv_internal.h"
#include "paged.h"

namespace fv {
namespace {

struct RopeParams {
    const void *q, *k;
    void *q_out, *k_out;
    long q_stride, k_stride, q_out_stride, k_out_stride;   // elements between tokens
    int heads, kv_heads, d, pairs, axes;
    const uint64_t* freq;
    const int* pair_axis;
    const int* positions;
    long tokens;
    float amplitude;
    int inverse;
    PagedDiv units;         // threads of a token in one piece of heads
    int turned;             // those of channels that are turned
    int per;                // heads a piece
};

// sin and cos of a fraction of a turn in units of 2^-64.
FV_DEV void turn_sincos(uint64_t turns, float& sin, float& cos) {
    const uint32_t t = (uint32_t)(turns >> 32) + ((uint32_t)turns >> 31);   // to the nearest 2^-32
    const uint32_t quarter = (t + 0x20000000u) >> 30;
    const float x = (float)(int)(t - (quarter << 30)) * (6.28318530717958647692f * 0x1p-32f), y = x * x;
    float s = __builtin_fmaf(y, 1.f / 362880.f, -1.f / 5040.f), c = __builtin_fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
    s = __builtin_fmaf(y, s, 1.f / 120.f), c = __builtin_fmaf(y, c, -1.f / 720.f);
    s = __builtin_fmaf(y, s, -1.f / 6.f), c = __builtin_fmaf(y, c, 1.f / 24.f);
    s = __builtin_fmaf(x * y, s, x), c = __builtin_fmaf(y, c, -0.5f);
    c = __builtin_fmaf(y, c, 1.f);
    sin = quarter & 1 ? c : s, cos = quarter & 1 ? s : c;
    sin = quarter & 2 ? -sin : sin, cos = (quarter + 1) & 2 ? -cos : cos;
}

// N channels: 16 bytes of bf16 or f32 in, as many or half or twice as many out.
template <bool IS16, int N>
FV_DEV void load_run(const void* base, long at, float (&x)[N]) {
    if constexpr (IS16) {
        static_assert(N == 8, "16 bytes");
        const u32x4 w = *reinterpret_cast<const u32x4*>((const uint16_t*)base + at);
#pragma unroll
        for (int i = 0; i < 4; i++) x[2 * i] = __builtin_bit_cast(float, w[i] << 16), x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
    } else {
        static_assert(N == 4, "16 bytes");
        const f32x4 w = *reinterpret_cast<const f32x4*>((const float*)base + at);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = w[i];
    }
}
template <bool IS16, int N>
FV_DEV void store_run(void* base, long at, const float (&x)[N]) {
    if constexpr (IS16) {
        typedef __attribute__((ext_vector_type(N))) float fv_n;
        typedef __attribute__((ext_vector_type(N))) __bf16 bf_n;
        fv_n v;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = x[i];
        *reinterpret_cast<bf_n*>((uint16_t*)base + at) = __builtin_convertvector(v, bf_n);
    } else {
#pragma unroll
        for (int h = 0; h < N; h += 4) *reinterpret_cast<f32x4*>((float*)base + at + h) = f32x4{x[h], x[h + 1], x[h + 2], x[h + 3]};
    }
}

// A thread has 16 bytes of a token's input a head (HALVES: and those of their partners), makes the angles of their pairs once, and goes through `per`
// heads of q and then k, four on their way at a time.
template <bool IN16, bool OUT16, bool HALVES>
__global__ __launch_bounds__(256) void rope_tokens_kernel(const RopeParams p) {
    constexpr int N = IN16 ? 8 : 4, kPairs = HALVES ? N : N / 2, kAtOnce = 4;
    const int id = blockIdx.x * 256 + threadIdx.x, token = paged_quot(id, p.units), unit = id - token * p.units.by;
    if (token >= p.tokens) return;
    const int all = p.heads + p.kv_heads, h0 = blockIdx.y * p.per, h1 = min(all, h0 + p.per);
    const bool turns = unit < p.turned;
    const int c0 = turns ? N * unit : 2 * p.pairs + N * (unit - p.turned), c1 = p.pairs + c0;   // (c1: HALVES' partners)
    const bool two = HALVES && turns;
    float c[kPairs], s[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; i++) c[i] = 1.f, s[i] = 0.f;
    if (turns) {
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const int pair = kPairs * unit + i;
            int axis = p.pair_axis ? p.pair_axis[pair] : 0;
            axis = (unsigned)axis < (unsigned)p.axes ? axis : 0;
            turn_sincos((uint64_t)(int64_t)p.positions[(long)token * p.axes + axis] * p.freq[pair], s[i], c[i]);
            s[i] = (p.inverse ? -s[i] : s[i]) * p.amplitude;
            c[i] *= p.amplitude;
        }
    }
    for (int h = h0; h < h1; h += kAtOnce) {
        float x[kAtOnce][N], y[kAtOnce][N];
#pragma unroll
        for (int j = 0; j < kAtOnce; j++) {
            const int head = min(h + j, h1 - 1);
            const bool is_k = head >= p.heads;
            const long from = token * (is_k ? p.k_stride : p.q_stride) + (long)(is_k ? head - p.heads : head) * p.d;
            load_run<IN16>(is_k ? p.k : p.q, from + c0, x[j]);
            if (two) load_run<IN16>(is_k ? p.k : p.q, from + c1, y[j]);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; j++) {
            if (turns) {
#pragma clang fp contract(off)
#pragma unroll
                for (int i = 0; i < kPairs; i++) {
                    const float a = HALVES ? x[j][i] : x[j][2 * i], b = HALVES ? y[j][i] : x[j][2 * i + 1];
                    const float u = a * c[i] - b * s[i], w = a * s[i] + b * c[i];
                    if constexpr (HALVES) x[j][i] = u, y[j][i] = w;
                    else x[j][2 * i] = u, x[j][2 * i + 1] = w;
                }
            }
            if (h + j < h1) {
                const bool is_k = h + j >= p.heads;
                const long to = token * (is_k ? p.k_out_stride : p.q_out_stride) + (long)(is_k ? h + j - p.heads : h + j) * p.d;
                store_run<OUT16>(is_k ? p.k_out : p.q_out, to + c0, x[j]);
                if (two) store_run<OUT16>(is_k ? p.k_out : p.q_out, to + c1, y[j]);
            }
        }
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace fv

extern "C" {

int fv_rope_frequencies(size_t pairs, double base, int scaling, double factor, double original, double low, double high, uint64_t* out) {
    if (!out) return fv_invalid("rope frequencies: null operand");
    if (pairs == 0 || pairs > 65536) return fv_invalid("rope frequencies: pairs");
    if (!(base >= 1.0) || !(base < 1e300)) return fv_invalid("rope frequencies: base must be 1 or more, and finite");
    if (scaling < 0 || scaling > 3) return fv_invalid("rope frequencies: scaling is 0 to 3");
    if (scaling != 0 && (!(factor >= 1.0) || !(factor < 1e9))) return fv_invalid("rope frequencies: factor must be 1 or more");
    if (scaling == 2 && pairs < 2) return fv_invalid("rope frequencies: a scaled base needs two pairs");
    if (scaling == 3 && (!(original > 0.0) || !(original < 1e18) || !(high > low) || !(high < 1e18) || !(low > -1e18)))
        return fv_invalid("rope frequencies: original must be positive and low below high");
    // (80 bits: a double's 53 leave a turn 2^-24 off at 2^31 positions)
    constexpr long double kTurn = 6.28318530717958647692528676655900577L;
    const long double n = (long double)pairs;
    long double b = base;
    if (scaling == 2) b *= powl(factor, n / (n - 1.0L));
    for (size_t i = 0; i < pairs; i++) {
        long double theta = powl(b, -(long double)i / n);
        if (scaling == 1) theta /= factor;
        if (scaling == 3) {
            const long double kept = std::min(1.0L, std::max(0.0L, (original * theta / kTurn - low) / (high - low)));
            theta *= kept + (1.0L - kept) / factor;
        }
        out[i] = (uint64_t)llrintl(ldexpl(theta / kTurn, 64));   // (theta is 1 at most: below 2^62)
    }
    return FV_OK;
}

int fv_rope_tokens(const void* q, size_t q_stride, void* q_out, size_t q_out_stride, size_t heads, const void* k, size_t k_stride, void* k_out,
                   size_t k_out_stride, size_t kv_heads, size_t d, int in_is_bf16, int out_is_bf16, const uint64_t* freq, const int32_t* pair_axis,
                   size_t pairs, const int32_t* positions, size_t axes, size_t tokens, float amplitude, int halves, int inverse, void* stream) {
    if (tokens == 0) return FV_OK;   // (empty arrays may have no address)
    if (!q || !q_out || !freq || !positions) return fv_invalid("rope tokens: null operand");
    if ((k == nullptr) != (k_out == nullptr)) return fv_invalid("rope tokens: keys without a place for the turned ones, or the reverse");
    if (heads == 0 || (k && kv_heads == 0)) return fv_invalid("rope tokens: no heads");
    if (!k) kv_heads = 0;
    if (d == 0 || d % 8 != 0 || d > 4096) return fv_decline("rope tokens: head dim must be a multiple of 8, 4096 at most");
    if (pairs == 0 || pairs % 8 != 0) return fv_decline("rope tokens: pairs must be a multiple of 8");
    if (2 * pairs > d) return fv_invalid("rope tokens: more pairs than channels");
    if (axes == 0 || axes > 4) return fv_invalid("rope tokens: 1 to 4 position axes");
    if (heads > 65535 || kv_heads > 65535) return fv_decline("rope tokens: too many heads");
    if (tokens > kMostRows) return fv_decline("rope tokens: too many tokens for one launch");
    if (!(amplitude > 0.f) || !(amplitude < 1e30f)) return fv_invalid("rope tokens: amplitude must be positive and finite");
    const size_t most = (size_t)INT_MAX / 4;
    struct {
        const void* at;
        size_t stride, heads;
    } const x[] = {{q, q_stride, heads}, {q_out, q_out_stride, heads}, {k, k_stride, kv_heads}, {k_out, k_out_stride, kv_heads}};
    for (size_t i = 0; i < (k ? 4 : 2); i++) {
        if (!fv::aligned16(x[i].at)) return fv_invalid("rope tokens: operands must be 16-byte aligned");
        if (x[i].stride < x[i].heads * d) return fv_invalid("rope tokens: tokens overlap (a stride below heads * d)");
        if (x[i].stride % 8 != 0 || x[i].stride > most) return fv_decline("rope tokens: strides must be multiples of 8 elements");
    }
    const bool same = (in_is_bf16 != 0) == (out_is_bf16 != 0);
    if ((q == q_out && (!same || q_stride != q_out_stride)) || (k && k == k_out && (!same || k_stride != k_out_stride)))
        return fv_invalid("rope tokens: in place only with one type and stride");
    fv::RopeParams p;
    p.q = q, p.k = k, p.q_out = q_out, p.k_out = k_out;
    p.q_stride = (long)q_stride, p.k_stride = (long)k_stride, p.q_out_stride = (long)q_out_stride, p.k_out_stride = (long)k_out_stride;
    p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.d = (int)d, p.pairs = (int)pairs, p.axes = (int)axes;
    p.freq = freq, p.pair_axis = pair_axis, p.positions = positions, p.tokens = (long)tokens;
    p.amplitude = amplitude, p.inverse = inverse != 0;
    const size_t run = in_is_bf16 ? 8 : 4, turned = (halves ? pairs : 2 * pairs) / run, units = turned + (d - 2 * pairs) / run, all = heads + kv_heads;
    if (tokens * units > (size_t)INT_MAX - 255) return fv_decline("rope tokens: too many tokens for one launch");
    // Heads of a thread: up to 16, so that the angles are a small part of its work; fewer where that leaves units without threads.
    const size_t wanted = (size_t)fv_compute_units() * 1024;
    size_t per = std::min<size_t>(all, 16);
    while (per > 1 && tokens * units * ((all + per - 1) / per) < wanted) per = (per + 1) / 2;
    per = std::max(per, (all + 65534) / 65535);   // (a grid's y is below 2^16)
    p.per = (int)per, p.turned = (int)turned, p.units = fv::paged_div(units);
    const dim3 blocks((unsigned)((tokens * units + 255) / 256), (unsigned)((all + per - 1) / per));
    if ((size_t)blocks.x * blocks.y >= (size_t)1 << 24) return fv_decline("rope tokens: too large for one launch");
    hipStream_t st = (hipStream_t)stream;
    fv::paged_pick(in_is_bf16 != 0, [&](auto i16) {
        fv::paged_pick(out_is_bf16 != 0, [&](auto o16) {
            fv::paged_pick(halves != 0, [&](auto h) {
                hipLaunchKernelGGL((fv::rope_tokens_kernel<i16(), o16(), h()>), blocks, dim3(256), 0, st, p);
            });
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "rope_tokens");
}

}  // extern "C"
