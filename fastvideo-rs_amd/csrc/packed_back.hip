// The gradients of attention over packed sequences (declarations: include/fv_sdpa_hip.h). With S = scale q k^T, P = e^(S - lse), D = sum(dout out)
// of every row (token, query head) and dS = P (dout v^T - D):
//     dv = P^T dout,    dk = scale dS^T q    (over the rows of all heads that share a key head),    dq = scale dS k.
//
// A scan makes -lse / scale and -D of every row. Then, in one launch, the keys' gradients, a workgroup for 128 keys that walks the rows which
// see them, and the queries', a workgroup for 128 rows that walks the keys: each accumulates in registers and writes once, so the sums have one
// order, no atomics and no cleared buffers. S and dP are made twice for that, seven products where five would do. To share them dq
// would go through memory as f32 sums of every key tile: 64 KB of atomic additions for 128 x 128 pairs of 128 channels, whose five products (21 MFLOP) take
// a unit 3.8 us at the rate of a large product (1399 TFLOP/s over 256 units): 4.4 TB/s over the card. That form is neither built nor measured; what
// stands against it is that the sums' order would change from call to call. Both statistics ride in the C operands of the products that
// make S and dP. Sums are f32. The products take bf16 operands (of f32 ones the matrix pipe does a sixteenth): P, dS and a dout in f32 are
// rounded for them, each by up to 2^-8 of itself.
#include <limits.h>

#include <algorithm>

#include "../../include/fv_sdpa_hip.h"
#include "packed.h"

namespace fv {
namespace {

constexpr int kRows = 128;   // of a workgroup of packed_dq_item, 32 a wave

// Which workgroup takes what, made on the device from the sequences' lengths (plan_pieces): the units of a key head, the longest first, each a
// piece of 128 rows or keys and a part [from, to) of the steps of its walk: tiles of 64 keys; of 32 rows. A walk longer than a slot's mean load is cut into
// shares, which leave f32 sums in places of 128 rows ([kv_heads][most_places][128][d or 2 d]) and are added by packed_sum_kernel.
struct BackUnit {
    int tile, from, to, place;         // place < 0: a whole walk; of a share: its place; kNoUnit: none. (Of a cut piece: `to` is its shares, `place` the first one's.)
    int start, count, k0, len, pos0;   // the sequence, as packed_seq has it
    FV_DEV PackedSeq seq() const { return {start, count, k0, len, pos0}; }
};
constexpr int kNoUnit = -2;
struct BackPlan {
    PagedPieces pieces;
    BackUnit *units, *cuts;   // (behind the last: kNoUnit)
    int2* scratch;       // every piece number's sequence and steps
    int most_units, most_cuts, most_places;   // of a key head
    float* places;
};

struct PackedBackParams {
    PackedBatch b;
    PackedMask mask;
    const uint16_t *q, *k, *v, *dout;
    long q_stride, k_stride, v_stride, dout_stride;   // bytes between tokens
    const float* stats;                               // [2][kv_heads][tokens * group]: -lse / scale; -D
    long stat_rows;                                   // of a plane
    void *dq, *dk, *dv;
    int grads_are_bf16;
    int heads, kv_heads;
    PagedDiv group;
    float scale, sl2;                                 // sl2 = scale * log2(e)
    PackedRuns runs;
    BackPlan rows, keys;                              // of packed_dq_item, of packed_dkv_item
};

// Chunk c of row r of a tile lies at chunk c ^ both_swz(r), so that a tile serves both kinds of operands without bank conflicts: the 8 rows of a
// transposed read lie at 8 different pairs of chunks, and the 16 lanes that a ds_read_b128 serves at once, rows 0 .. 3 and 12 .. 15 of one chunk
// and 4 .. 11 of its neighbour, at 16 different chunks (64 channels: 8, in two halves of a line): with the rows' pairs in order
// rows 8 .. 15 take the other chunk of the pairs of rows 4 .. 7, 0 .. 3.
template <int D>
FV_DEV int both_swz(int r) {
    return D == 128 ? (((r & 7) ^ ((r >> 1) & 4)) << 1 | ((r >> 3) & 1)) : ((((r >> 1) & 3) ^ ((r >> 2) & 2)) << 1 | ((r >> 3) & 1));
}
template <int D>
FV_DEV TileReadBases both_bases(int lane) {
    using G = TileGeo<D>;
    const int q4 = lane >> 4, i16 = lane & 15, r = 4 * q4 + (i16 >> 2);
    return {i16 * G::kRow + ((both_swz<D>(i16) ^ q4) << 4), r * G::kRow + ((both_swz<D>(r) ^ ((i16 & 3) >> 1)) << 4) + 8 * (i16 & 1)};
}

// The rows of a sequence, counted (token, head of the group), that see a key: [lo, hi), hi INT_MAX where that is to the last.
struct KeySight {
    int lo, hi;
};
template <class Mask>
FV_DEV KeySight key_sight(const Mask& m, const PackedSeq& s, int key, int group) {
    if (!m.causal) return {0, 0x7fffffff};
    const int bt = m.block_tokens.by, block = paged_quot(key, m.block_tokens);
    const long lo = (long)block * bt - s.pos0, hi = m.window > 0 && block >= m.sink ? (long)block * bt + (long)m.window * bt - s.pos0 : s.count;
    KeySight k;
    k.lo = (int)min(max(lo, 0L), (long)s.count) * group;
    k.hi = hi >= s.count ? 0x7fffffff : (int)max(hi, 0L) * group;
    return k;
}
// The rows of a sequence that see one key, [lo, hi): their weight is 1 and their dS nothing, exactly, where dP - D would leave the rounding of `out`.
// packed_dkv_item loads zeros for their queries and -lse / scale (scores of 0, a weight of 1, no part in dk), packed_dq_item stores zeros. By
// token those are the first token's (under a window of one, without a sink, all); by blocks those of a last block of one key under such a window.
// (Others see one of the keys that max_k keeps and are not among these: their dS is what dP - D leaves.)
template <class Mask>
FV_DEV KeySight single_rows(const Mask& m, const PackedSeq& s, int group) {
    const bool alone = m.window == 1 && m.sink == 0;
    if (!m.causal) return {0, s.len == 1 ? 0x7fffffff : 0};
    const int bt = m.block_tokens.by;
    if (bt > 1 && !(s.len == 1 || (alone && s.len - paged_quot(s.len, m.block_tokens) * bt == 1))) return {0, 0};
    const int pos = bt == 1 ? 0 : s.len - 1;   // (a row at a negative position sees none)
    const int first = (int)min(max((long)pos - s.pos0, 0L), (long)s.count), behind = bt == 1 && alone ? s.count : (int)min(max((long)pos + 1 - s.pos0, 0L), (long)s.count);
    return {first * group, behind * group};
}

// packed_dkv_item: a workgroup's keys, the rows of a step, and its LDS: V's operands | 2 x (q, dout) | 2 x (-lse / scale, -D).
constexpr int kKeys = 128, kStep = 32;
template <int D>
struct KeyForm {
    static constexpr int kHalf = kStep * 2 * D;   // bytes of a step's q, or dout
    static constexpr int kFrags = D / 16, kSteps = 4 * kFrags * 1024, kStats = kSteps + 4 * kHalf, kLds = kStats + 2 * 256;
};
// The steps [from, to) that some key of [first, last] is seen by.
struct RowWalk {
    int from, to;
};
template <class Mask>
FV_DEV RowWalk row_walk(const Mask& m, const PackedSeq& s, int first, int last, int group) {
    const int rows = s.count * group;
    const KeySight a = key_sight(m, s, first, group), b = key_sight(m, s, last, group);
    return {a.lo / kStep, (min(rows, max(a.hi, b.hi)) + kStep - 1) / kStep};
}

// The steps of a piece's walk.
template <bool KEYS>
FV_DEV int back_steps(const PackedBackParams& p, const PackedSeq& sq, int tile) {
    if constexpr (KEYS) {
        const int key0 = tile * kKeys;
        if (key0 >= sq.len) return -1;
        const RowWalk w = row_walk(p.mask, sq, key0, min(key0 + kKeys, sq.len) - 1, p.group.by);
        return max(w.to - w.from, 0);
    } else {
        const int rows = sq.count * p.group.by, row0 = tile * kRows;
        if (row0 >= rows) return -1;
        return packed_walk(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group)).n;
    }
}
// Steps below which no walk is cut; a step of a row's walk (64 keys x 128 rows, three products) in steps of a key's (128 keys x 32 rows, four); what a
// share costs: with S steps in all, shares of A steps take A steps' time and leave S / A places, each 1 / kShares of a step for its traffic (of 128
// keys 256 KB, of 128 rows 128), which is least for A = sqrt(S / kShares). (Five sequences of some 100 rows and keys, 16 heads on one: 50 -> 32 us.)
constexpr int kLeastKeys = 4, kLeastRows = 3, kSharesKeys = 10, kSharesRows = 25;
constexpr float kRowStep = 1.5f;
// The first piece of a sequence; the sequence and the steps of a piece (steps < 0: of an unused number).
template <bool KEYS>
FV_DEV long plan_first(const PackedBackParams& p, const PackedBatch& b, const BackPlan& plan, int seq) {
    constexpr int R = KEYS ? kKeys : kRows;
    const PackedKeys kb = {b.k_start, b.seqs, b.k_tokens};
    return KEYS ? paged_first_piece<R>(plan.pieces, kb, 1, seq) : paged_first_piece<R>(plan.pieces, b, p.group.by, seq);
}
template <bool KEYS>
FV_DEV int2 plan_piece(const PackedBackParams& p, const PackedBatch& b, const BackPlan& plan, int n) {
    constexpr int R = KEYS ? kKeys : kRows;
    auto first_of = [&](int seq) { return plan_first<KEYS>(p, b, plan, seq); };
    int seq = 0;
    if (plan.pieces.tiles.by) {
        seq = paged_quot(n, plan.pieces.tiles);
    } else {
        int behind = b.seqs;   // the last of sequences seq .. behind - 1 whose first piece is no later
        while (behind - seq > 1) {
            const int mid = seq + (behind - seq) / 2;
            if (first_of(mid) <= n) seq = mid;
            else behind = mid;
        }
    }
    const long tile = n - first_of(seq);
    return {seq, tile < 0 || tile > 0x7fffffff / R ? -1 : back_steps<KEYS>(p, packed_seq(b, seq), (int)tile)};
}
// One workgroup makes a plan: the walks' lengths; their sum, and from it the length past which a walk is cut into equal shares; the units
// sorted by their lengths into 64 classes, longest first (in a class in any order: it changes no result). By itself the order of the pieces left slots idle
// for a third of the time (one clip of 7 frames, 12 heads, 1032 pieces on 512 slots) or for two thirds (a window with a sink, whose keys all rows see).
// The rows' walks are cut past their mean load of a slot, the keys' past the mean load of both kinds, since the rows' units come behind and fill
// what is idle (21 prompts of up to 702 tokens, 32 / 8 heads: 227 -> 206 us).
template <bool KEYS>
FV_DEV void plan_pieces(const PackedBackParams& p, const BackPlan& plan, int slots) {
    constexpr int kClasses = 64, kHeld = 1024;
    __shared__ unsigned long long sum, others;
    __shared__ int longest, units[kClasses], cuts, places, total, held[2][kHeld];
    const int tid = threadIdx.x, numbers = plan.pieces.n.by;
    if (tid == 0) sum = 0, others = 0, longest = 0, cuts = 0, places = 0;
    if (tid < kClasses) units[tid] = 0;
    PackedBatch b = p.b;
    if (b.seqs < kHeld) {   // (a search makes a chain of reads: from LDS)
        for (int i = tid; i <= b.seqs; i += 256) held[0][i] = b.q_start[i], held[1][i] = b.k_start[i];
        b.q_start = held[0], b.k_start = held[1];
    }
    __syncthreads();
    unsigned long long mine = 0, theirs = 0;
    int most = 0;
    const int rows_at = (numbers + 63) & ~63;   // (the other kind in the same turns, by other waves)
    for (int n = tid; n < (KEYS ? rows_at + p.rows.pieces.n.by : numbers); n += 256) {
        if (n < numbers) {
            const int2 x = plan_piece<KEYS>(p, b, plan, n);
            plan.scratch[n] = x;
            mine += (unsigned long long)max(x.y, 0), most = max(most, x.y);
        } else if (n >= rows_at) {
            theirs += (unsigned long long)max(plan_piece<false>(p, b, p.rows, n - rows_at).y, 0);
        }
    }
    atomicAdd(&sum, mine);
    atomicMax(&longest, most);
    if constexpr (KEYS) atomicAdd(&others, theirs);
    __syncthreads();
    const float all = (float)sum * (float)p.kv_heads, behind = KEYS ? kRowStep * (float)others * (float)p.kv_heads : 0.f;
    const float least = __builtin_sqrtf(all / (KEYS ? kSharesKeys : kSharesRows));
    const int load = (int)min(max(max((all + behind) / (float)slots, least) + 1.f, (float)(KEYS ? kLeastKeys : kLeastRows)), 1e9f);
    auto shares_of = [&](int steps) { return steps > load ? (steps + load - 1) / load : 1; };
    const float per_step = (float)kClasses / (float)(min(longest, load) + 1);
    auto class_of = [&](int chunk) { return kClasses - 1 - min((int)((float)chunk * per_step), kClasses - 1); };   // 0: the longest
    auto chunk_of = [](int steps, int shares) { return shares == 1 ? steps : (steps + shares - 1) / shares; };
    for (int n = tid; n < numbers; n += 256) {
        const int steps = plan.scratch[n].y;
        if (steps < 0) continue;
        const int k = shares_of(steps);
        atomicAdd(&units[class_of(chunk_of(steps, k))], k);
    }
    __syncthreads();
    if (tid < kClasses) {   // (a wave)
        const int n = units[tid];
        int upto = n;
#pragma unroll
        for (int d = 1; d < kClasses; d <<= 1) {
            const int x = __shfl_up(upto, d, 64);
            upto += tid >= d ? x : 0;
        }
        units[tid] = upto - n;
        if (tid == kClasses - 1) total = upto;
    }
    __syncthreads();
    for (int n = tid; n < numbers; n += 256) {
        const int2 x = plan.scratch[n];
        if (x.y < 0) continue;
        const PackedSeq sq = packed_seq(b, x.x);
        const int k = shares_of(x.y), chunk = chunk_of(x.y, k), tile = (int)(n - plan_first<KEYS>(p, b, plan, x.x));
        int u = atomicAdd(&units[class_of(chunk)], k), place = -1;
        if (k > 1) {
            const int c = atomicAdd(&cuts, 1);
            place = atomicAdd(&places, k);
            if (c < plan.most_cuts) plan.cuts[c] = BackUnit{tile, 0, k, place, sq.start, sq.count, sq.k0, sq.len, sq.pos0};
        }
        for (int i = 0; i < k; i++, u++)
            if (u < plan.most_units) plan.units[u] = BackUnit{tile, i * chunk, min(x.y, (i + 1) * chunk), place < 0 ? -1 : place + i, sq.start, sq.count, sq.k0, sq.len, sq.pos0};
    }
    __syncthreads();
    for (int u = total + tid; u < plan.most_units; u += 256) plan.units[u].place = kNoUnit;
    for (int c = cuts + tid; c < plan.most_cuts; c += 256) plan.cuts[c].place = kNoUnit;
}

// D / 8 threads a row (token, head); OUT16, DOUT16: bf16 bits. An f32 gradient is kept as bf16 bits in `rounded` [tokens, heads, d].
// FEW, in calls whose rows see 64 keys at most: one that sees up to kFew has sum_j p_j (dout . v_j) in place of sum(dout out). The rounding of `out` is up to
// 2^-8 of it, which is as much as what dS is made of where few keys share a row and one has most of its weight (dq and dk of sequences of 2 to 4 tokens
// were 0.0051 of their size off, are 0.0032). Everywhere the search for a row's sequence would cost 24 us of 1990 (5 prompts of up to 6000), where such rows are few.
constexpr int kFew = 8, kFewKeys = 64;
template <int D, bool OUT16, bool DOUT16, bool FEW>
__global__ __launch_bounds__(256, 8) void packed_stats_kernel(const PackedBackParams p, const void* dout, const void* out, const float* lse, float* stats, uint16_t* rounded,
                                                           long rows, float inv_scale, int slots) {
    if (blockIdx.x < 2) {   // (the first two: the plans)
        if (blockIdx.x == 0) plan_pieces<true>(p, p.keys, slots);
        else plan_pieces<false>(p, p.rows, slots);
        return;
    }
    constexpr int kPer = D / 8;
    const int c = threadIdx.x % kPer, heads = p.heads;
    const long row = (long)(blockIdx.x - 2) * (256 / kPer) + threadIdx.x / kPer, tokens = p.b.tokens;
    const PagedDiv group = p.group;
    if (row >= rows) return;
    auto eight = [&](const void* at, auto is16, float (&x)[8]) {
        if constexpr (is16()) {
            const u32x4 w = *reinterpret_cast<const u32x4*>((const uint16_t*)at + row * D + 8 * c);
#pragma unroll
            for (int i = 0; i < 4; i++) x[2 * i] = __builtin_bit_cast(float, w[i] << 16), x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f32x4 w = *reinterpret_cast<const f32x4*>((const float*)at + row * D + 8 * c + 4 * h);
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * h + i] = w[i];
            }
        }
    };
    float g[8], o[8], sum = 0.f;
    eight(dout, std::integral_constant<bool, DOUT16>{}, g);
    eight(out, std::integral_constant<bool, OUT16>{}, o);
    if constexpr (!DOUT16) {
        f32x8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = g[i];
        const bf16x8 y = __builtin_convertvector(x, bf16x8);
        *reinterpret_cast<bf16x8*>(rounded + row * D + 8 * c) = y;
        x = __builtin_convertvector(y, f32x8);   // (the gradient that the products see)
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] = x[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) sum = __builtin_fmaf(g[i], o[i], sum);
#pragma unroll
    for (int s = 1; s < kPer; s <<= 1) sum += __shfl_xor(sum, s, 64);
    const long t = row / heads;
    const int h = (int)(row - t * heads), kvh = paged_quot(h, group);
    const float l = lse[row];
    if constexpr (FEW) {
        // the last sequence that begins no later than the token: for the wave's first by scalar reads, from there on by the lane
        using Starts = const __attribute__((address_space(4))) int*;
        const int t0 = __builtin_amdgcn_readfirstlane((int)t);
        int seq = 0;
        for (int behind = p.b.seqs; behind - seq > 1;) {
            const int mid = seq + (behind - seq) / 2;
            if (((Starts)p.b.q_start)[mid] <= t0) seq = mid;
            else behind = mid;
        }
        if (seq + 1 < p.b.seqs && p.b.q_start[seq + 1] <= t) {
            seq++;
            for (int behind = p.b.seqs; behind - seq > 1;) {
                const int mid = seq + (behind - seq) / 2;
                if (p.b.q_start[mid] <= t) seq = mid;
                else behind = mid;
            }
        }
        const PackedSeq sq = packed_seq(p.b, seq);
        const int in = (int)t - sq.start;
        const PagedSight sees = in >= 0 && in < sq.count ? packed_sight(p.mask, sq.pos0 + in, sq.len) : PagedSight{0, 0, 0};
        const int band = max(sees.lo, sees.a), keys = sees.a + max(sees.hi - band, 0);
        if (keys > 1 && keys <= kFew) {
            auto bits = [](const uint16_t* at, float (&x)[8]) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
                for (int i = 0; i < 4; i++) x[2 * i] = __builtin_bit_cast(float, w[i] << 16), x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
            };
            float qx[8];
            bits((const uint16_t*)((const uint8_t*)p.q + t * p.q_stride) + h * D + 8 * c, qx);
            sum = 0.f;
#pragma unroll 1
            for (int j = 0; j < keys; j += 2) {
                float s[2], dp[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int x = min(j + u, keys - 1);
                    const long key = sq.k0 + (x < sees.a ? x : band + x - sees.a);
                    float kx[8], vx[8];
                    bits((const uint16_t*)((const uint8_t*)p.k + key * p.k_stride) + kvh * D + 8 * c, kx);
                    bits((const uint16_t*)((const uint8_t*)p.v + key * p.v_stride) + kvh * D + 8 * c, vx);
                    s[u] = dp[u] = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) s[u] = __builtin_fmaf(qx[i], kx[i], s[u]), dp[u] = __builtin_fmaf(g[i], vx[i], dp[u]);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
#pragma unroll
                    for (int x = 1; x < kPer; x <<= 1) s[u] += __shfl_xor(s[u], x, 64), dp[u] += __shfl_xor(dp[u], x, 64);
                    if (j + u < keys) sum += fast_exp2((s[u] - l * inv_scale) * p.sl2) * dp[u];
                }
            }
        }
    }
    if (c == 0) {
        float* at = stats + ((long)kvh * tokens + t) * group.by + (h - kvh * group.by);
        at[0] = l == neg_inf() ? l : -l * inv_scale;
        at[rows] = -sum;
    }
}

// ---- the keys' gradients ---------------------------------------------------------------------------------------------

// A wave's part in a step of 32 rows at `qt` and `gt` (q and dout), `cut`: with keys that rows do not see, whose scores become -inf. The
// products, two to a unit that shares an operand read: S = Q K^T - lse / scale, 16 rows after 16; dP = dO V^T - D; dV^T += dO^T P; dK^T += Q^T dS.
// The vector work lies in their shadow: a 16x16x32 product holds the matrix pipe for four instructions' time, of which two others of the same wave cost
// nothing (measured, with one wave a SIMD: 8.1 ns a product with none, 8.7 with two multiplications, 10.3 with three; an exponential counts for two). So the
// exponentials of the first 16 rows run under the scores of the others and dP, dS under dV. With the softmax by itself between dP and dV: 5 to 6 %
// slower. Operands are read three units ahead: one, 15 % slower; four need registers that are not there.
template <int D>
FV_DEV void key_step(const lds_u8* qt, const lds_u8* gt, const lds_u8* vt, const lds_u8* stat, const TileReadBases& rb, const bf16x8 (&kf)[D / 32][2],
                     f32x4 (&dk)[D / 16][2], f32x4 (&dv)[D / 16][2], float sl2, bool cut, const KeySight (&mine)[2], int row0) {
    using G = TileGeo<D>;
    constexpr int kNK = D / 32, U = 2 * kNK, kUnits = 4 * U, kAhead = 3;
    const int lane = threadIdx.x & 63, q4 = lane >> 4;
    bf16x8 a[kUnits], b[kNK][2];        // a unit's operand; V's
    int read_k = rb.k, read_v = rb.v;   // (pinned: the addresses made from them would take registers over the whole loop)
    asm volatile("" : "+v"(read_k), "+v"(read_v));
    auto issue = [&](int u) {
        if (u < U) {              // Q, 16 rows u / kNK
            a[u] = lds_read_b128(qt + (read_k ^ ((u % kNK) << 6)) + (u / kNK) * 16 * G::kRow);
        } else if (u < 2 * U) {   // dO, 16 rows u % 2 of d chunk (u - U) / 2, and before the first V's
            const int dc = (u - U) >> 1, x = u & 1;
            if (x == 0) {
#pragma unroll
                for (int g = 0; g < 2; g++) b[dc][g] = lds_read_b128(vt + (2 * dc + g) * 1024 + lane * 16);
            }
            a[u] = lds_read_b128(gt + (read_k ^ (dc << 6)) + x * 16 * G::kRow);
        } else {                  // dO^T, then Q^T, 16 channels u % U
            a[u] = read_v_frag<D>((u < 3 * U ? gt : qt) + (read_v ^ ((u % U) << 5)));
        }
    };
    f32x4 s[2][2], dp[2][2], init_s[2], init_d[2];   // [16 rows][16 keys]; what their sums start from
    bf16x8 pb[2], ds[2];       // the second products' operands: of 32 rows, those of both blocks that the lane has
    // Vector work k of 16 scores, of the first 16 rows first: the lane's rows i of keys g.
    auto score = [&](int k) { s[k >> 3][(k >> 2) & 1][k & 3] = fast_exp2(s[k >> 3][(k >> 2) & 1][k & 3] * sl2); };
    auto weigh = [&](int k) { dp[k >> 3][(k >> 2) & 1][k & 3] *= s[k >> 3][(k >> 2) & 1][k & 3]; };
    auto round = [&](const f32x4 (&from)[2][2], bf16x8 (&to)[2], int c) {   // pair c of 8
        const int g = c >> 2, x = (c >> 1) & 1, i = 2 * (c & 1);
        const bf16x2 y = __builtin_convertvector((f32x2{from[x][g][i], from[x][g][i + 1]}), bf16x2);
        to[g][4 * x + i] = y[0], to[g][4 * x + i + 1] = y[1];
    };
    auto stat_rows = [&](int x, int which) { return *reinterpret_cast<const __attribute__((address_space(3))) f32x4*>(stat + 128 * which + (16 * x + 4 * q4) * 4); };
    auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
    auto hide = [&](int x) {
        if (!cut) return;
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int r = row0 + 16 * x + 4 * q4;
            const unsigned bits = below(mine[g].hi - r) & ~below(mine[g].lo - r);
#pragma unroll
            for (int i = 0; i < 4; i++) s[x][g][i] = (bits >> i) & 1 ? s[x][g][i] : neg_inf();
        }
    };
    auto gap = [&](auto n) {   // behind product n
        if constexpr (n() == 2 * U - 6 || n() == 2 * U - 4) {
            constexpr int x = (n() - 2 * U + 6) / 2;
            init_d[x] = stat_rows(x, 1);
        }
        if constexpr (n() == U + 1) hide(0);
        if constexpr (n() == 2 * U + 1) hide(1);
        static_for<16>([&](auto k) {
            if constexpr (n() == U + 2 + k() * U / 8) score(k());
            if constexpr (n() == 4 * U + 2 + k() * U / 16) weigh(k());
            if constexpr (k() < 8 && n() == 3 * U + 2 + k() * U / 16) round(s, pb, k());
            if constexpr (k() < 8 && n() == 5 * U + 2 + k() * U / 16) round(dp, ds, k());
        });
    };
#pragma unroll
    for (int u = 0; u < kAhead; u++) issue(u);
#pragma unroll
    for (int x = 0; x < 2; x++) init_s[x] = stat_rows(x, 0);
    __builtin_amdgcn_s_setprio(1);
    static_for<2 * kUnits>([&](auto at) {
        constexpr int u = at() / 2, g = at() & 1;
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (u < U) s[u / kNK][g] = mfma16(a[u], kf[u % kNK][g], u % kNK == 0 ? init_s[u / kNK] : s[u / kNK][g]);
        else if constexpr (u < 2 * U) dp[u & 1][g] = mfma16(a[u], b[(u - U) >> 1][g], u < U + 2 ? init_d[u & 1] : dp[u & 1][g]);
        else if constexpr (u < 3 * U) dv[u % U][g] = mfma16(a[u], pb[g], dv[u % U][g]);
        else dk[u % U][g] = mfma16(a[u], ds[g], dk[u % U][g]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (g == 0 && u + kAhead < kUnits) issue(u + kAhead);
        gap(at);
    });
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
}

// 128 keys of one (sequence, key head), 32 a wave, over steps of 32 rows of q and dout that pass through LDS, two buffers each (three, a step's
// rows on their way for two: 6 to 9 % slower). A lane has two keys (columns lane % 16 and 16 + lane % 16 of its wave's): S and dP [rows x keys]
// come out of the products in the layout that the second ones take P and dS in, and dV^T, dK^T [d x keys] stay in 128 registers (64 at 64 channels). K's operands stay in registers, V's in LDS as they are read: an operand is read once for two products, and an LDS
// read a product costs nothing (at two waves a SIMD 1706 and 1715 TFLOP/s of 16x16x32 with half a ds_read_b128 each and one).
template <int D>
FV_DEV void packed_dkv_item(const PackedBackParams& p, const int wave, const int lane, const int block) {
    using G = TileGeo<D>;
    using F = KeyForm<D>;
    constexpr int kNO = D / 16, kNK = D / 32, kHalf = F::kHalf;
    constexpr int kLoads = kHalf / 4096;   // of a wave: its part of a step's q
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    lds_u8* smem = (lds_u8*)smem_raw;
    const int q4 = lane >> 4, i16 = lane & 15;
    const PackedSlot at = packed_slot(p.runs, block, p.keys.most_units);
    if (at.head < 0) return;
    const BackUnit unit = p.keys.units[at.number];
    if (unit.place == kNoUnit) return;
    const int kvh = at.head, group = p.group.by;
    const PackedSeq sq = unit.seq();
    const int key0 = unit.tile * kKeys;
    const int rows = sq.count * group, last = min(key0 + kKeys, sq.len) - 1;
    const RowWalk walk = row_walk(p.mask, sq, key0, last, group);
    const int e0 = walk.from + unit.from, e1 = min(walk.to, walk.from + unit.to);

    // the wave's keys: rows that see some of them, rows that see all; the lane's two
    const int wkey = key0 + 32 * wave;
    const bool idle = wkey >= sq.len;
    KeySight mine[2], some = {0, 0}, all = {0, 0};
#pragma unroll
    for (int g = 0; g < 2; g++) mine[g] = key_sight(p.mask, sq, min(wkey + 16 * g + i16, sq.len - 1), group);
    if (!idle) {
        const int to = min(wkey + 31, last), early = (int)min((long)p.mask.sink * p.mask.block_tokens.by, (long)to);   // (of the keys past the sink the first is seen for the shortest)
        const KeySight a = key_sight(p.mask, sq, wkey, group), b = key_sight(p.mask, sq, to, group);
        some = {a.lo, max(a.hi, b.hi)}, all = {b.lo, key_sight(p.mask, sq, max(wkey, early), group).hi};
    }
    const KeySight single = single_rows(p.mask, sq, group);
    const uint16_t *kbase = p.k + kvh * D, *vbase = p.v + kvh * D;
    const unsigned lds0 = (unsigned)(size_t)smem;
    // V: the wave's operands, 1 KB each: the lane's 16 bytes of key i16 (+ 16) and chunk 4 dc + q4
    bf16x8 kf[kNK][2];
    {
        const u32x4 vd = packed_rows(vbase, sq.k0 + wkey, p.v_stride, min(sq.len - wkey, 32), G::kRow);
        const unsigned at = (unsigned)i16 * (unsigned)p.v_stride + 16u * q4;
#pragma unroll
        for (int f = 0; f < F::kFrags; f++) {
            const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds0 + (wave * F::kFrags + f) * 1024)), off = at + (f & 1) * 16u * (unsigned)p.v_stride + (f >> 1) * 64;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(m0), "v"(off), "s"(vd) : "memory");
        }
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int key = min(wkey + 16 * g + i16, sq.len - 1);   // (past the last: the last again, not stored)
        const uint16_t* at = (const uint16_t*)((const uint8_t*)kbase + (long)(sq.k0 + key) * p.k_stride) + 8 * q4;
#pragma unroll
        for (int dk = 0; dk < kNK; dk++) kf[dk][g] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(at + 32 * dk));
    }
    // Steps are loaded from the walk's last to its first: their rows' tokens t0 .. and the h0 heads of t0 before them, and where t0 and the statistics lie, go
    // back by 32 rows a step. (The same from the step's number, 50 scalar instructions in a row, cost 13 to 17 % of the time.) Row x of a step is token t0 + dt,
    // dt = (h0 + x) / group, of numbers below group + 32. Rows lie in the order of their addresses, so those behind the last are cut off by the
    // descriptor (zeros); only the walk's last step has any.
    const int back = kStep / group, back_heads = kStep - back * group;   // tokens and heads of 32 rows
    const unsigned mul = 65536u / (unsigned)group + 1, qstep = (unsigned)p.q_stride - (unsigned)(group * G::kRow), gstep = (unsigned)p.dout_stride - (unsigned)(group * G::kRow);
    auto row_dt = [&](int x) { return group >= 32 ? (x >= group ? 1 : 0) : (int)((unsigned)x * mul >> 16); };
    const int r_last = (e1 - 1) * kStep, t_last = paged_quot(r_last, p.group);
    int h0 = r_last - t_last * group;
    const uint8_t* qb = (const uint8_t*)p.q + (long)(sq.start + t_last) * p.q_stride + (long)kvh * group * G::kRow;
    const uint8_t* gb = (const uint8_t*)p.dout + (long)(sq.start + t_last) * p.dout_stride + (long)kvh * group * G::kRow;
    const float* sb = p.stats + (wave & 1) * p.stat_rows + ((long)kvh * p.b.tokens + sq.start) * group + r_last;
    unsigned qo[kLoads], go[kLoads];
    auto offsets = [&]() {
#pragma unroll
        for (int it = 0; it < kLoads; it++) {
            const int rr = (wave * kLoads + it) * G::kRowsPerDma + lane / G::kChunks, x = h0 + rr, dt = row_dt(x);
            const unsigned in = (unsigned)(x * G::kRow) + ((unsigned)((lane % G::kChunks) ^ both_swz<D>(rr)) << 4);
            qo[it] = (unsigned)dt * qstep + in, go[it] = (unsigned)dt * gstep + in;
        }
    };
    offsets();
    unsigned q_bytes, g_bytes, s_bytes;
    {
        const int n = max(min(rows - r_last, kStep), 1), end = h0 + n - 1, dt_end = row_dt(end);   // the last row
        q_bytes = (unsigned)dt_end * qstep + (unsigned)(end + 1) * G::kRow, g_bytes = (unsigned)dt_end * gstep + (unsigned)(end + 1) * G::kRow, s_bytes = n * 4u;
    }
    int r_at = r_last;   // the step's first row
    auto load = [&](int buf) {
        const bool some_single = r_at < single.hi && r_at + kStep > single.lo;
        const u32x4 qd = plane_descriptor(qb, q_bytes), gd = plane_descriptor(gb, g_bytes);
        const unsigned at = lds0 + F::kSteps + buf * 2 * kHalf + wave * (kHalf / 4);
#pragma unroll
        for (int it = 0; it < kLoads; it++) {
            const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(at + it * 1024)), m1 = m0 + kHalf;
            unsigned from = qo[it];
            if (some_single) {
                const int r = r_at + (wave * kLoads + it) * G::kRowsPerDma + lane / G::kChunks;
                from = r >= single.lo && r < single.hi ? 0x80000000u : from;   // (past the descriptor: zeros)
            }
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
                         "s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds"
                         :: "s"(m0), "s"(m1), "v"(from), "v"(go[it]), "s"(qd), "s"(gd) : "memory");
        }
        if (wave < 2) {   // (32 floats, -lse / scale or -D)
            const u32x4 sd = plane_descriptor(sb, s_bytes);
            const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds0 + F::kStats + buf * 256 + wave * 128));
            const bool none = wave == 0 && r_at + lane >= single.lo && r_at + lane < single.hi;
            if (lane < 32) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" :: "s"(m0), "v"(none ? 0x80000000u : lane * 4u), "s"(sd) : "memory");
        }
        r_at -= kStep;
        q_bytes = g_bytes = 0x80000000u, s_bytes = 128;
        h0 -= back_heads;
        const bool more = h0 < 0;
        h0 += more ? group : 0;
        qb -= (long)(back + more) * p.q_stride, gb -= (long)(back + more) * p.dout_stride, sb -= kStep;
        if (back_heads != 0) offsets();
    };
    const TileReadBases rb = both_bases<D>(lane);
    f32x4 dv[kNO][2], dk[kNO][2];
#pragma unroll
    for (int db = 0; db < kNO; db++)
#pragma unroll
        for (int g = 0; g < 2; g++) dv[db][g] = dk[db][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float sl2 = p.sl2;

    // (The walk goes backwards: under a causal mask every piece ends at the sequence's last row, so that workgroups that begin together go through the same
    // rows, which an L2 then holds.)
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): K's operands, on every path, or the compiler waits for them, and so for the steps' loads, in the loop
    if (e0 < e1) {
        load(0);
        wait_vmcnt<0>();
        block_barrier();
    }
    int buf = 0;
#pragma unroll 1
    for (int e = e1 - 1; e >= e0; e--) {
        if (e - 1 >= e0) load(buf ^ 1);
        if ((e + 1) * kStep > some.lo && e * kStep < some.hi && !idle) {
            const lds_u8* step = smem + F::kSteps + buf * 2 * kHalf;
            const bool cut = e * kStep < all.lo || (e + 1) * kStep > all.hi;
            key_step<D>(step, step + kHalf, smem + wave * F::kFrags * 1024, smem + F::kStats + buf * 256, rb, kf, dk, dv, sl2, cut, mine, e * kStep);
        }
        buf ^= 1;
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<0>();
        block_barrier();   // the next step resident; this one's read by every wave
        __builtin_amdgcn_sched_barrier(0);
    }
    auto dst_key = [&](int key) { return ((size_t)(sq.k0 + key) * p.kv_heads + kvh) * D; };
#pragma unroll
    for (int db = 0; db < kNO; db++)
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) dk[db][g][i] *= p.scale;
    if (unit.place < 0 && p.grads_are_bf16) {   // (through the wave's own LDS of its fragments, which are of no more use)
        if (idle) return;
        lds_u8* my = smem + wave * F::kFrags * 1024;
        bf16x4 y[kNO][2];
        auto rounded = [&](const f32x4 (&x)[kNO][2]) {
#pragma unroll
            for (int db = 0; db < kNO; db++)
#pragma unroll
                for (int g = 0; g < 2; g++) y[db][g] = __builtin_convertvector(x[db][g], bf16x4);
        };
        rounded(dk);
        packed_store_rows<D>(my, y, lane, [&](int r) -> uint16_t* { return wkey + r < sq.len ? (uint16_t*)p.dk + dst_key(wkey + r) : nullptr; });
        rounded(dv);
        packed_store_rows<D>(my, y, lane, [&](int r) -> uint16_t* { return wkey + r < sq.len ? (uint16_t*)p.dv + dst_key(wkey + r) : nullptr; });
        return;
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int key = wkey + 16 * g + i16;
        if (key >= sq.len) continue;
        float* part = p.keys.places + (((size_t)kvh * p.keys.most_places + max(unit.place, 0)) * kKeys + (key - key0)) * 2 * D;
        float *to_dk = unit.place >= 0 ? part : (float*)p.dk + dst_key(key), *to_dv = unit.place >= 0 ? part + D : (float*)p.dv + dst_key(key);
#pragma unroll
        for (int db = 0; db < kNO; db++) {
            *reinterpret_cast<f32x4*>(to_dk + 16 * db + 4 * q4) = dk[db][g];
            *reinterpret_cast<f32x4*>(to_dv + 16 * db + 4 * q4) = dv[db][g];
        }
    }
}

// ---- the queries' gradients ------------------------------------------------------------------------------------------

// A wave's part in a tile of 64 keys at `kt` and `vt`, `cut`: with keys that rows do not see (key0: the tile's first). In halves of 32 keys, two
// products to a unit: S^T = K Q^T - lse / scale and dP^T = V dO^T - D of the one, of the other, dQ^T += K^T dS of the one, of the other, with the vector work
// in their shadow, as in key_step: the exponentials under dP, dS of a half under what follows it.
template <int D>
FV_DEV void row_step(const lds_u8* kt, const lds_u8* vt, const TileReadBases& rb, const bf16x8 (&qf)[D / 32][2], const bf16x8 (&gf)[D / 32][2],
                     const f32x4 (&s_init)[2], const f32x4 (&d_init)[2], f32x4 (&dq)[D / 16][2], float sl2, bool cut, const PagedSight& mine, int key0) {
    using G = TileGeo<D>;
    constexpr int kNK = D / 32, U = 2 * kNK, kAll = 6 * U, kAhead = 3;
    const int q4 = (threadIdx.x >> 4) & 3;
    bf16x8 a[kAll];
    int read_k = rb.k, read_v = rb.v;
    asm volatile("" : "+v"(read_k), "+v"(read_v));
    auto issue = [&](int n) {
        if (n < 4 * U) {   // K, V of the first half, K, V of the second: 16 keys (n % U) / kNK, d chunk n % kNK
            const int half = n / (2 * U), x = n % U / kNK;
            a[n] = lds_read_b128((n / U & 1 ? vt : kt) + (read_k ^ ((n % kNK) << 6)) + (32 * half + 16 * x) * G::kRow);
        } else {           // K^T, 16 channels n % U
            a[n] = read_v_frag<D>(kt + (read_v ^ ((n % U) << 5)) + 32 * (n / U - 4) * G::kRow);
        }
    };
    f32x4 s[2][2][2], dp[2][2][2];   // [half][16 keys][16 rows]
    bf16x8 ds[2][2];
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int g = 0; g < 2; g++) s[half][x][g] = s_init[g];
    if (cut) {
        const unsigned m[3] = {(unsigned)mine.a, (unsigned)mine.lo, (unsigned)mine.hi};
        int both[3][2];   // the even rows of 16 lanes hold block 0's, the odd ones block 1's
#pragma unroll
        for (int x = 0; x < 3; x++) {
            const auto r = __builtin_amdgcn_permlane16_swap(m[x], m[x], false, false);
            both[x][0] = (int)r[0];
            both[x][1] = (int)r[1];
        }
        auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const int at = key0 + 32 * half + 16 * x + 4 * q4;
                    const unsigned bits = below(both[0][g] - at) | (below(both[2][g] - at) & ~below(both[1][g] - at));
#pragma unroll
                    for (int i = 0; i < 4; i++) s[half][x][g][i] = (bits >> i) & 1 ? s[half][x][g][i] : neg_inf();
                }
    }
    auto score = [&](int half, int k) {   // k: of 16, the first 16 keys first
        const int x = k >> 3, g = (k >> 2) & 1, i = k & 3;
        s[half][x][g][i] = fast_exp2(s[half][x][g][i] * sl2);
    };
    auto weigh = [&](int half, int k) {
        const int x = k >> 3, g = (k >> 2) & 1, i = k & 3;
        dp[half][x][g][i] *= s[half][x][g][i];
    };
    auto round = [&](int half, int c) {   // pair c of 8
        const int g = c >> 2, x = (c >> 1) & 1, i = 2 * (c & 1);
        const bf16x2 y = __builtin_convertvector((f32x2{dp[half][x][g][i], dp[half][x][g][i + 1]}), bf16x2);
        ds[half][g][4 * x + i] = y[0], ds[half][g][4 * x + i + 1] = y[1];
    };
    auto gap = [&](auto n) {   // behind product n
        static_for<32>([&](auto i) {
            constexpr int half = i() / 16, k = i() % 16, m = n() - 4 * U * half;
            if constexpr (m == U + 2 + k * U / 8) score(half, k);
            if constexpr (m == (k < 8 ? 3 * U + 2 + k * U / 16 : 4 * U + 2 + (k - 8) * U / 16)) weigh(half, k);
            if constexpr (k < 8 && m == 4 * U + 2 + U / 2 + k * U / 16) round(half, k);
        });
    };
#pragma unroll
    for (int n = 0; n < kAhead; n++) issue(n);
    __builtin_amdgcn_s_setprio(1);
    static_for<2 * kAll>([&](auto at) {
        constexpr int n = at() / 2, g = at() & 1, half = n / (2 * U), x = n % U / kNK, dc = n % kNK;
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (n >= 4 * U) dq[n % U][g] = mfma16(a[n], ds[n / U - 4][g], dq[n % U][g]);
        else if constexpr (n / U & 1) dp[half][x][g] = mfma16(a[n], gf[dc][g], dc == 0 ? d_init[g] : dp[half][x][g]);
        else s[half][x][g] = mfma16(a[n], qf[dc][g], s[half][x][g]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (g == 0 && n + kAhead < kAll) issue(n + kAhead);
        gap(at);
    });
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
}

// 128 rows of one (sequence, key head), 32 a wave, over tiles of 64 keys in LDS, two buffers for K and for V. Q and dO stay in registers; S^T =
// K Q^T and dP^T = V dO^T leave the scores of two rows in a lane, dS the operand of dQ^T += K^T dS, whose K is the
// same tile read across.
template <int D>
FV_DEV void packed_dq_item(const PackedBackParams& p, const int wave, const int lane, const int block) {
    using G = TileGeo<D>;
    constexpr int kNO = D / 16, kNK = D / 32, kTile = G::kTile, kIter = TileDma<4, D>::ITER, kUnits = kIter / 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    lds_u8* smem = (lds_u8*)smem_raw;
    const int q4 = lane >> 4, i16 = lane & 15;
    const PackedSlot at = packed_slot(p.runs, block, p.rows.most_units);
    if (at.head < 0) return;
    const BackUnit unit = p.rows.units[at.number];
    if (unit.place == kNoUnit) return;
    const int kvh = at.head, group = p.group.by;
    const PackedSeq sq = unit.seq();
    const int rows = sq.count * group, row0 = unit.tile * kRows;
    const int wrow = row0 + 32 * wave;
    const bool idle = wrow >= rows;
    bf16x8 qf[kNK][2], gf[kNK][2];
    f32x4 s_init[2], d_init[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = min(wrow + 16 * g + i16, rows - 1), t = paged_quot(r, p.group);   // (past the last: the last again, not stored)
        const long in = (long)(kvh * group + r - t * group) * G::kRow + 16 * q4;
        const uint8_t* q = (const uint8_t*)p.q + (long)(sq.start + t) * p.q_stride + in;
        const uint8_t* go = (const uint8_t*)p.dout + (long)(sq.start + t) * p.dout_stride + in;
#pragma unroll
        for (int dk = 0; dk < kNK; dk++) {
            qf[dk][g] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(q + 64 * dk));
            gf[dk][g] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(go + 64 * dk));
        }
        const float* at = p.stats + ((long)kvh * p.b.tokens + sq.start) * group + r;
        const float nlse = at[0], nd = at[p.stat_rows];
#pragma unroll
        for (int i = 0; i < 4; i++) s_init[g][i] = nlse, d_init[g][i] = nd;
    }
    const PackedWalk w = packed_walk(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group));
    const int e0 = unit.from, e1 = min(w.n, unit.to);
    const KeySight single = single_rows(p.mask, sq, group);
    const float sl2 = p.sl2;

    PagedSight all_see = {0x7fffffff, 0, 0x7fffffff}, mine = {0, 0, 0};
    if (!idle) {
        all_see = packed_all(p.mask, sq, paged_quot(wrow, p.group), paged_quot(min(wrow + 32, rows) - 1, p.group));
        mine = packed_sight(p.mask, sq.pos0 + paged_quot(min(wrow + (lane & 31), rows - 1), p.group), sq.len);
    }
    const PackedWhole whole = packed_whole(w, all_see);
    unsigned koff[kIter], voff[kIter];
    packed_offsets<D>(koff, (unsigned)p.k_stride, wave, lane, [](int r) { return both_swz<D>(r); });
    packed_offsets<D>(voff, (unsigned)p.v_stride, wave, lane, [](int r) { return both_swz<D>(r); });
    const uint16_t *kbase = p.k + kvh * D, *vbase = p.v + kvh * D;
    const unsigned slot = (unsigned)(size_t)smem + wave * kIter * 1024;
    PackedRun krun(kbase, p.k_stride, sq, w, e0), vrun(vbase, p.v_stride, sq, w, e0);
    auto load = [&](int buf) {
        const u32x4 kd = krun.rows(G::kRow), vd = vrun.rows(G::kRow);
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            packed_issue(kd, koff[2 * u], koff[2 * u + 1], slot + buf * kTile + u * 2048);
            packed_issue(vd, voff[2 * u], voff[2 * u + 1], slot + (2 + buf) * kTile + u * 2048);
        }
        krun.next(), vrun.next();
    };
    if (e0 < e1) load(0);   // (the first keys and values on their way beside the operands')
    const TileReadBases rb = both_bases<D>(lane);
    f32x4 dq[kNO][2];
#pragma unroll
    for (int db = 0; db < kNO; db++) dq[db][0] = dq[db][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the operands and statistics, on every path (as above), and the first tile
    if (e0 < e1) block_barrier();
#pragma unroll 1
    for (int e = e0; e < e1; e++) {
        const int buf = (e - e0) & 1;
        if (e + 1 < e1) load(buf ^ 1);
        if (!idle) {
            const lds_u8* kt = smem + buf * kTile;
            row_step<D>(kt, kt + 2 * kTile, rb, qf, gf, s_init, d_init, dq, sl2, !whole.tile(e), mine, w.key(e));
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<0>();
        block_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    auto dst_row = [&](int r) {
        const int t = paged_quot(r, p.group);
        return ((size_t)(sq.start + t) * p.heads + kvh * group + (r - t * group)) * D;
    };
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = wrow + 16 * g + i16;
        const bool alone = r >= single.lo && r < single.hi;
#pragma unroll
        for (int db = 0; db < kNO; db++)
#pragma unroll
            for (int i = 0; i < 4; i++) dq[db][g][i] = alone ? 0.f : dq[db][g][i] * p.scale;
    }
    if (unit.place < 0 && p.grads_are_bf16) {   // (through the tiles' LDS, which every wave has read)
        if (idle) return;
        bf16x4 y[kNO][2];
#pragma unroll
        for (int db = 0; db < kNO; db++)
#pragma unroll
            for (int g = 0; g < 2; g++) y[db][g] = __builtin_convertvector(dq[db][g], bf16x4);
        packed_store_rows<D>(smem + wave * (32 * G::kRow), y, lane, [&](int r) -> uint16_t* { return wrow + r < rows ? (uint16_t*)p.dq + dst_row(wrow + r) : nullptr; });
        return;
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = wrow + 16 * g + i16;
        if (r >= rows) continue;
        float* to = unit.place >= 0 ? p.rows.places + (((size_t)kvh * p.rows.most_places + max(unit.place, 0)) * kRows + (r - row0)) * D : (float*)p.dq + dst_row(r);
#pragma unroll
        for (int db = 0; db < kNO; db++) *reinterpret_cast<f32x4*>(to + 16 * db + 4 * q4) = dq[db][g];
    }
}

// The keys' units first, then the rows', whose shorter walks fill what the last of the keys' leave idle.
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_back_kernel(const PackedBackParams p, int key_blocks) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, block = blockIdx.x;
    if (block < key_blocks) packed_dkv_item<D>(p, wave, lane, block);
    else packed_dq_item<D>(p, wave, lane, block - key_blocks);
}

// The shares of cut walks, added in their order: D / 4 threads a row of dq or (KEYS) twice as many a key, dk and dv, `per` rows or keys a workgroup. (The
// grid is that of as many cut pieces as there may be.)
template <int D, bool KEYS>
FV_DEV void packed_sum(const PackedBackParams& p, int block, int per) {
    constexpr int kPiece = KEYS ? kKeys : kRows, kWide = KEYS ? 2 * D : D, kPer = kWide / 4, kSum = 256 / kPer, kAtOnce = 4;
    const BackPlan& plan = KEYS ? p.keys : p.rows;
    const int c = threadIdx.x % kPer, parts = kPiece / per, item = block / parts, in0 = (block - item * parts) * per;
    const int number = item / p.kv_heads, kvh = item - number * p.kv_heads, group = p.group.by;
    const BackUnit cut = plan.cuts[number];
    if (cut.place == kNoUnit) return;
    const PackedSeq sq = cut.seq();
    const int rows = KEYS ? sq.len : sq.count * group;
    for (int in = in0 + threadIdx.x / kPer; in < in0 + per; in += kSum) {
        const int r = cut.tile * kPiece + in;
        if (r >= rows) return;
        const float* part = plan.places + (((size_t)kvh * plan.most_places + cut.place) * kPiece + in) * kWide + 4 * c;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < cut.to; s += kAtOnce) {
            f32x4 y[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) y[u] = *reinterpret_cast<const f32x4*>(part + (size_t)min(s + u, cut.to - 1) * kPiece * kWide);
#pragma unroll
            for (int u = 0; u < kAtOnce; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] += s + u < cut.to ? y[u][i] : 0.f;
        }
        void* out;
        size_t dst;
        if constexpr (KEYS) {
            out = 4 * c < D ? p.dk : p.dv;
            dst = ((size_t)(sq.k0 + r) * p.kv_heads + kvh) * D + 4 * c % D;
        } else {
            const int t = paged_quot(r, p.group);
            out = p.dq;
            dst = ((size_t)(sq.start + t) * p.heads + kvh * group + (r - t * group)) * D + 4 * c;
        }
        if (p.grads_are_bf16) *reinterpret_cast<bf16x4*>((uint16_t*)out + dst) = __builtin_convertvector(x, bf16x4);
        else *reinterpret_cast<f32x4*>((float*)out + dst) = x;
    }
}
template <int D>
__global__ __launch_bounds__(256) void packed_sum_kernel(const PackedBackParams p, int key_blocks, int per) {
    const int block = blockIdx.x;
    if (block < key_blocks) packed_sum<D, true>(p, block, per);
    else packed_sum<D, false>(p, block - key_blocks, per);
}

// A call's plans and its workspace. With a walk cut where it passes the mean load of a slot there are no more shares past the first of a piece
// than slots, and no more places than twice as many; walks of no more than `least` steps are not cut.
struct BackParts {
    size_t stats = 0, rounded = 0, bytes = 0;   // bytes from the workspace's start
    int slots;
    struct Plan {
        PagedPieces pieces;
        size_t units, cuts, places, units_at, cuts_at, scratch_at, places_at;
    } keys, rows;
    BackParts(const PackedCall& c, bool round) {
        auto take = [this](size_t n) {
            const size_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        slots = (c.d == 64 ? 3 : 2) * fv_compute_units();
        const size_t group = c.heads / c.kv_heads;
        auto plan = [&](Plan& x, const PagedPieces& pieces, size_t steps, size_t least, size_t place_bytes) {
            x.pieces = pieces;
            const size_t n = (size_t)pieces.n.by, more = steps > least ? std::min((size_t)slots / c.kv_heads + 1, n * (steps / least)) : 0;
            x.units = n + more, x.cuts = std::min(n, more), x.places = 2 * more;
            x.units_at = take(x.units * sizeof(BackUnit)), x.cuts_at = take(x.cuts * sizeof(BackUnit)), x.scratch_at = take(n * 8);
            x.places_at = take(x.places * c.kv_heads * place_bytes);
        };
        stats = take(c.tokens * c.heads * 8);
        if (round) rounded = take(c.tokens * c.heads * c.d * 2);
        plan(keys, paged_pieces(kKeys, c.seqs, c.k_tokens, c.max_k, 1), (c.max_q * group + kStep - 1) / kStep, kLeastKeys, kKeys * c.d * 8);
        plan(rows, paged_pieces(kRows, c.seqs, c.tokens, c.max_q, group), fv_packed_key_steps(c, kRows), kLeastRows, kRows * c.d * 4);
    }
    static BackPlan on_device(const Plan& x, uint8_t* ws) {
        return {x.pieces, (BackUnit*)(ws + x.units_at), (BackUnit*)(ws + x.cuts_at), (int2*)(ws + x.scratch_at), (int)x.units, (int)x.cuts,
                (int)x.places, (float*)(ws + x.places_at)};
    }
};
// (the one kernel here that takes more than 64 KB)
hipError_t packed_prepare() {
    static std::atomic<unsigned long long> done{0};
    static_assert(KeyForm<64>::kLds <= 65536, "no attribute");
    return fv_set_max_lds_once((const void*)packed_back_kernel<128>, KeyForm<128>::kLds, done);
}

}  // namespace
}  // namespace fv

extern "C" hipError_t fv_internal_init_packed(void) { return fv::packed_prepare(); }

extern "C" {

size_t fv_packed_attention_backward_workspace_bytes(int dout_is_bf16, size_t heads, size_t kv_heads, size_t d, size_t seqs, size_t q_tokens,
                                                    size_t k_tokens, size_t max_q, size_t max_k, int causal, size_t block_tokens, size_t window,
                                                    size_t sink) {
    const PackedCall c = {heads, kv_heads, d, seqs, q_tokens, k_tokens, std::min(max_q, q_tokens), std::min(max_k, k_tokens), nullptr, nullptr, 1.f, causal,
                          block_tokens, window, sink};
    return fv_packed_sizes(c) ? fv::BackParts(c, !dout_is_bf16).bytes : 0;
}

int fv_packed_attention_backward(const void* dout, int dout_is_bf16, const uint16_t* q, size_t q_stride, const uint16_t* k, size_t k_stride,
                                 const uint16_t* v, size_t v_stride, const void* out, int out_is_bf16, const float* lse, void* dq, void* dk, void* dv,
                                 int grads_are_bf16, size_t heads, size_t kv_heads, size_t d, const int32_t* q_start, const int32_t* k_start,
                                 size_t seqs, size_t q_tokens, size_t k_tokens, size_t max_q, size_t max_k, float scale, int causal,
                                 size_t block_tokens, size_t window, size_t sink, void* workspace, size_t workspace_bytes, void* stream) {
    const PackedCall c = {heads, kv_heads, d, seqs, q_tokens, k_tokens, std::min(max_q, q_tokens), std::min(max_k, k_tokens), q_start, k_start, scale,
                          causal, block_tokens, window, sink};
    if (seqs == 0 || (c.max_q == 0 && c.max_k == 0)) return FV_OK;   // (no unit to launch; empty arrays may have no address)
    PackedOperand x[9];
    size_t n = 0;
    if (q_tokens > 0) {
        const size_t s = heads * d;
        x[n++] = {q, q_stride, heads}, x[n++] = {dout, s, heads}, x[n++] = {out, s, heads}, x[n++] = {dq, s, heads};
        if (!lse) return fv_invalid("packed attention backward: null operand");
    }
    if (k_tokens > 0) x[n++] = {k, k_stride, kv_heads}, x[n++] = {v, v_stride, kv_heads}, x[n++] = {dk, kv_heads * d, kv_heads}, x[n++] = {dv, kv_heads * d, kv_heads};
    const int rc = fv_packed_args("packed attention backward", c, x, n, workspace);
    if (rc != FV_OK) return rc;
    const fv::BackParts parts(c, !dout_is_bf16);
    if (!workspace || workspace_bytes < parts.bytes) return fv_invalid("packed attention backward: workspace too small");
    const size_t rows = q_tokens * heads, stat_blocks = (rows + 2048 / d - 1) / (2048 / d) + 2;
    // Rows or keys of a workgroup of the sums: 8 where few pieces may be cut (their shares are many, a wait each), up to 32 where the grid would hold
    // thousands without work (8 us of 25000).
    size_t per = 8;
    static_assert(fv::kRows == fv::kKeys, "one number for both");
    while (per < 32 && kv_heads * (parts.rows.cuts + parts.keys.cuts) * (fv::kRows / per) > 4096) per *= 2;
    const size_t sum_rows = kv_heads * parts.rows.cuts * (fv::kRows / per), sum_keys = kv_heads * parts.keys.cuts * (fv::kKeys / per);
    constexpr size_t kMost = (size_t)1 << 24;   // (a launch holds fewer than 2^32 work-items)
    if (kv_heads * (parts.rows.units + parts.keys.units) >= kMost / 2 || stat_blocks >= kMost || sum_rows + sum_keys >= kMost)
        return fv_decline("packed attention backward: too large for one launch");
    uint8_t* ws = (uint8_t*)workspace;
    fv::PackedBackParams p;
    p.b = {q_start, k_start, (int)seqs, (int)q_tokens, (int)k_tokens, (int)c.max_q, (int)c.max_k};
    p.mask = fv_packed_mask(c);
    p.q = q, p.k = k, p.v = v, p.dout = dout_is_bf16 ? (const uint16_t*)dout : (const uint16_t*)(ws + parts.rounded);
    p.q_stride = (long)q_stride * 2, p.k_stride = (long)k_stride * 2, p.v_stride = (long)v_stride * 2, p.dout_stride = (long)(heads * d * 2);
    p.stats = (const float*)(ws + parts.stats), p.stat_rows = (long)(q_tokens * heads);
    p.dq = dq, p.dk = dk, p.dv = dv, p.grads_are_bf16 = grads_are_bf16 != 0;
    p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = fv::paged_div(heads / kv_heads);
    p.scale = scale, p.sl2 = (float)((double)scale * 1.4426950408889634);
    p.runs = fv::packed_runs(kv_heads, causal != 0);
    p.keys = fv::BackParts::on_device(parts.keys, ws), p.rows = fv::BackParts::on_device(parts.rows, ws);
    const bool few = c.max_k <= (size_t)fv::kFewKeys || (causal && window > 0 && (window + sink) * block_tokens <= (size_t)fv::kFewKeys);   // (below 2^32 each)
    hipStream_t st = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    fv::paged_pick(d == 128, [&](auto d128) {
        constexpr int D = d128() ? 128 : 64;
        fv::paged_pick(out_is_bf16 != 0, [&](auto o16) {
            fv::paged_pick(dout_is_bf16 != 0, [&](auto g16) {
                fv::paged_pick(few, [&](auto f) {
                    hipLaunchKernelGGL((fv::packed_stats_kernel<D, o16(), g16(), f()>), dim3((unsigned)stat_blocks), dim3(256), 0, st, p, dout, out, lse,
                                       (float*)(ws + parts.stats), (uint16_t*)(ws + parts.rounded), (long)rows, (float)(1.0 / (double)scale), parts.slots);
                });
            });
        });
        const size_t key_blocks = fv::packed_blocks(p.runs, parts.keys.units), row_blocks = fv::packed_blocks(p.runs, parts.rows.units);
        if (D == 128) e = fv::packed_prepare();
        if (e != hipSuccess) return;
        hipLaunchKernelGGL((fv::packed_back_kernel<D>), dim3((unsigned)(key_blocks + row_blocks)), dim3(256), fv::KeyForm<D>::kLds, st, p, (int)key_blocks);
        if (sum_keys + sum_rows > 0) hipLaunchKernelGGL((fv::packed_sum_kernel<D>), dim3((unsigned)(sum_keys + sum_rows)), dim3(256), 0, st, p, (int)sum_keys, (int)per);
    });
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "packed_attention_backward");
}

}  // extern "C"
