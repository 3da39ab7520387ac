// The gradients of attention over packed sequences (declarations: include/fv_sdpa_hip.h). With S = scale q k^T, P = e^(S - lse), D = sum(dout out)
// of every row (token, query head) and dS = P (dout v^T - D):
//     dv = P^T dout,    dk = scale dS^T q    (over the rows of all heads that share a key head),    dq = scale dS k.
//
// Three launches. A scan makes -lse / scale and -D of every row. Then the keys' gradients, a workgroup for 128 keys that walks the rows which
// see them, and the queries', a workgroup for 128 rows that walks the keys: each accumulates in registers and writes once, so the sums have one
// order, no atomics and no cleared buffers. S and dP are made twice for that (seven products where five would do): to share them dq
// would go through memory as f32 sums of every key tile, 512 B a row and 128 keys, at 0.19 us of matrix work for 128 x 128 pairs of five
// products an atomic stream of 64 KB, in an order that changes. Both statistics ride in the C operands of the products that
// make S and dP. Sums are f32; P and dS are rounded to bf16 for the second products (2^-9 of each).
#include <limits.h>

#include <algorithm>

#include "../../include/fv_sdpa_hip.h"
#include "packed.h"

namespace fv {
namespace {

constexpr int kRows = 128;       // rows of a workgroup of packed_dq_kernel, keys of one of packed_dkv_kernel: 32 a wave
constexpr int kStepRows = 32;    // rows a step of packed_dkv_kernel takes

struct PackedBackParams {
    PackedBatch b;
    PackedMask mask;
    const uint16_t *q, *k, *v, *dout;
    long q_stride, k_stride, v_stride, dout_stride;   // bytes between tokens
    const f32x2* stats;                               // [kv_heads][tokens * group]: -lse / scale, -D
    void *dq, *dk, *dv;
    int grads_are_bf16;
    int heads, kv_heads;
    PagedDiv group;
    float scale, sl2;                                 // sl2 = scale * log2(e)
    PagedPieces row_pieces, key_pieces;
    PackedItems row_items, key_items;
    int row_chunk, key_chunk;                         // steps of a walk that a workgroup takes: tiles of 64 keys; of 32 rows
    // shares of walks longer than that, f32: [shares][128 rows of every piece][d]; [shares][128 keys of every piece][2][d]
    float *part_dq, *part_dkv;
    long part_rows, part_keys;
};

// Chunk c of row r of a tile lies at chunk c ^ both_swz(r): the 16 rows of a ds_read_b128 lie at 16 different chunks (64 channels: 8, in two halves
// of a line) and the 8 rows of a transposed read at 8 different pairs of them, so a tile serves both kinds of operands without conflicts.
template <int D>
FV_DEV int both_swz(int r) { return D == 128 ? ((r & 7) << 1 | ((r >> 3) & 1)) : (((r >> 1) & 3) << 1 | ((r >> 3) & 1)); }
template <int D>
FV_DEV TileReadBases both_bases(int lane) {
    using G = TileGeo<D>;
    const int q4 = lane >> 4, i16 = lane & 15, r = 4 * q4 + (i16 >> 2);
    return {i16 * G::kRow + ((both_swz<D>(i16) ^ q4) << 4), r * G::kRow + ((both_swz<D>(r) ^ ((i16 & 3) >> 1)) << 4) + 8 * (i16 & 1)};
}

// D / 8 threads a row (token, head); OUT16, DOUT16: bf16 bits. An f32 gradient is kept as bf16 bits in `rounded` [tokens, heads, d].
template <int D, bool OUT16, bool DOUT16>
__global__ __launch_bounds__(256) void packed_stats_kernel(const void* dout, const void* out, const float* lse, f32x2* stats, uint16_t* rounded, long rows,
                                                           long tokens, int heads, PagedDiv group, float inv_scale) {
    constexpr int kPer = D / 8;
    const int c = threadIdx.x % kPer;
    const long row = (long)blockIdx.x * (256 / kPer) + threadIdx.x / kPer;
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
    if (c == 0) {
        const long t = row / heads;
        const int h = (int)(row - t * heads), kvh = paged_quot(h, group);
        const float l = lse[row];
        stats[((long)kvh * tokens + t) * group.by + (h - kvh * group.by)] = f32x2{l == neg_inf() ? l : -l * inv_scale, -sum};
    }
}

// ---- the keys' gradients ---------------------------------------------------------------------------------------------

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
// The steps [from, to) of kStepRows rows that some key of [first, last] is seen by.
struct RowWalk {
    int from, to;
};
template <class Mask>
FV_DEV RowWalk row_walk(const Mask& m, const PackedSeq& s, int first, int last, int group) {
    const int rows = s.count * group;
    const KeySight a = key_sight(m, s, first, group), b = key_sight(m, s, last, group);
    return {a.lo / kStepRows, (min(rows, max(a.hi, b.hi)) + kStepRows - 1) / kStepRows};
}

// 128 keys of one (sequence, key head), 32 a wave, over steps of 32 rows of q and dout that pass through LDS, two buffers each. A lane has
// two keys (columns lane % 16 and 16 + lane % 16 of its wave's): S and dP [rows x keys] come out of the products in the layout that the second ones
// take P and dS in, and dV^T, dK^T [d x keys] stay in 128 registers (64 at 64 channels). K's operands stay in registers, V's in LDS, which
// has room for it: a product's operands are read once for two, and an LDS read a product costs nothing (at two waves a SIMD 1706
// and 1715 TFLOP/s of 16x16x32 with half a ds_read_b128 each and one).
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_dkv_kernel(const PackedBackParams p) {
    using G = TileGeo<D>;
    constexpr int kNO = D / 16, kNK = D / 32, kHalf = kStepRows * G::kRow;   // bytes of a step's q, or dout
    constexpr int kLoads = kHalf / 4096;                                       // of a wave: its part of a step's q
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    lds_u8* smem = (lds_u8*)smem_raw;
    // V | 2 x (q, dout) | 2 x stats
    constexpr int kSteps = kRows * G::kRow, kStats = kSteps + 4 * kHalf;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q4 = lane >> 4, i16 = lane & 15;
    const PackedItem item = packed_item(p.key_items, blockIdx.x);
    if (item.head < 0) return;
    const int kvh = item.head, group = p.group.by;
    const PackedKeys kb = {p.b.k_start, p.b.seqs, p.b.k_tokens};
    const PagedPiece piece = paged_piece<kRows>(p.key_pieces, kb, 1, item.piece);   // (a sequence's first keys, which most rows see, first)
    const PackedSeq sq = packed_seq(p.b, piece.seq);
    const int key0 = piece.tile * kRows;
    if (key0 >= sq.len) return;
    const int rows = sq.count * group, last = min(key0 + kRows, sq.len) - 1;
    const RowWalk walk = row_walk(p.mask, sq, key0, last, group);
    const int e0 = walk.from + item.share * p.key_chunk, e1 = min(walk.to, e0 + p.key_chunk);
    if (item.share > 0 && e0 >= e1) return;
    const bool split = walk.to - walk.from > p.key_chunk;

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
    const uint16_t *kbase = p.k + kvh * D, *vbase = p.v + kvh * D;
    // V: the wave's 32 rows into its part of LDS
    const unsigned lds0 = (unsigned)(size_t)smem;
    {
        constexpr int kIter = 32 * G::kRow / 1024;
        const u32x4 vd = packed_rows(vbase, sq.k0 + wkey, p.v_stride, min(sq.len - wkey, 32), G::kRow);
#pragma unroll
        for (int it = 0; it < kIter; it += 2) {
            unsigned off[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int r = (it + x) * G::kRowsPerDma + lane / G::kChunks, c = lane % G::kChunks;
                off[x] = (unsigned)r * (unsigned)p.v_stride + ((unsigned)(c ^ both_swz<D>(r)) << 4) - x * 1024u;
            }
            packed_issue(vd, off[0], off[1], lds0 + wave * 32 * G::kRow + it * 1024);
        }
    }
    bf16x8 kf[kNK][2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int key = wkey + 16 * g + i16;
        const uint16_t* at = (const uint16_t*)((const uint8_t*)kbase + (long)(sq.k0 + key) * p.k_stride) + 8 * q4;
#pragma unroll
        for (int dk = 0; dk < kNK; dk++) {
            u32x4 x = {0u, 0u, 0u, 0u};
            if (key < sq.len) x = *reinterpret_cast<const u32x4*>(at + 32 * dk);
            kf[dk][g] = __builtin_bit_cast(bf16x8, x);
        }
    }
    // A step's rows into buffer `buf`: each wave loads 8 rows of q and of dout, the first one the statistics.
    auto load = [&](int e, int buf) {
        const int r0 = e * kStepRows, t0 = paged_quot(r0, p.group);
        const uint8_t* qb = (const uint8_t*)p.q + (long)(sq.start + t0) * p.q_stride + (long)kvh * group * G::kRow;
        const uint8_t* gb = (const uint8_t*)p.dout + (long)(sq.start + t0) * p.dout_stride + (long)kvh * group * G::kRow;
        const u32x4 qd = plane_descriptor(qb, 0x80000000u), gd = plane_descriptor(gb, 0x80000000u);
        const unsigned at = lds0 + kSteps + buf * 2 * kHalf + wave * (kHalf / 4);
#pragma unroll
        for (int it = 0; it < kLoads; it++) {
            const int rr = (wave * kLoads + it) * G::kRowsPerDma + lane / G::kChunks, r = r0 + rr, t = paged_quot(r, p.group);
            const unsigned in = (unsigned)((r - t * group) * G::kRow) + ((unsigned)((lane % G::kChunks) ^ both_swz<D>(rr)) << 4);
            const bool none = r >= rows;   // (past the range: zeros)
            const unsigned qo = none ? 0x80000000u : (unsigned)(t - t0) * (unsigned)p.q_stride + in, go = none ? 0x80000000u : (unsigned)(t - t0) * (unsigned)p.dout_stride + in;
            const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(at + it * 1024)), m1 = m0 + kHalf;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
                         "s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds"
                         :: "s"(m0), "s"(m1), "v"(qo), "v"(go), "s"(qd), "s"(gd) : "memory");
        }
        if (wave == 0) {
            const u32x4 sd = plane_descriptor(p.stats + ((long)kvh * p.b.tokens + sq.start) * group + r0, (unsigned)min(rows - r0, kStepRows) * 8u);
            const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds0 + kStats + buf * 256));
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" :: "s"(m0), "v"(lane * 4), "s"(sd) : "memory");
        }
    };
    const TileReadBases rb = both_bases<D>(lane);
    f32x4 dv[kNO][2], dk[kNO][2];
#pragma unroll
    for (int db = 0; db < kNO; db++)
#pragma unroll
        for (int g = 0; g < 2; g++) dv[db][g] = dk[db][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float sl2 = p.sl2;

    if (e0 < e1) {
        load(e0, 0);
#pragma unroll
        for (int x = 0; x < kNK; x++) asm volatile("" : "+v"(kf[x][0]), "+v"(kf[x][1]));   // (waited for here)
        wait_vmcnt<0>();
        block_barrier();
    }
#pragma unroll 1
    for (int e = e0; e < e1; e++) {
        const int buf = (e - e0) & 1, r0 = e * kStepRows;
        if (e + 1 < e1) load(e + 1, buf ^ 1);
        if (r0 + kStepRows > some.lo && r0 < some.hi && !idle) {
            const lds_u8* qt = smem + kSteps + buf * 2 * kHalf;
            const lds_u8* gt = qt + kHalf;
            const lds_u8* vt = smem + wave * 32 * G::kRow;
            const lds_u8* stat = smem + kStats + buf * 256;
            f32x4 s[2][2], dp[2][2];   // [16 rows][16 keys]
            // S = Q K^T - lse / scale and dP = dO V^T - D: a group is two operands of 16 rows (dP: and two of keys) for four products
            constexpr int kN1 = 2 * kNK, kAhead = 2;
            bf16x8 f[kN1][2], fv[kN1][2];
            auto issue1 = [&](int i, int x) {
                const int at = (rb.k ^ ((i >> 1) << 6)) + x * 16 * G::kRow;
                if (i & 1) f[i][x] = lds_read_b128(gt + at), fv[i][x] = lds_read_b128(vt + at);
                else f[i][x] = lds_read_b128(qt + at);
            };
            f32x4 init_s[2], init_d[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const auto* at = reinterpret_cast<const __attribute__((address_space(3))) f32x4*>(stat + (16 * x + 4 * q4) * 8);
                const f32x4 a = at[0], b = at[1];
                init_s[x] = f32x4{a[0], a[2], b[0], b[2]};
                init_d[x] = f32x4{a[1], a[3], b[1], b[3]};
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < kAhead; i++) issue1(i, 0), issue1(i, 1);
#pragma unroll
            for (int i = 0; i < kN1; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int x = j >> 1, g = j & 1;
                    __builtin_amdgcn_sched_barrier(0);
                    if (i & 1) dp[x][g] = mfma16(f[i][x], fv[i][g], i < 2 ? init_d[x] : dp[x][g]);
                    else s[x][g] = mfma16(f[i][x], kf[i >> 1][g], i < 2 ? init_s[x] : s[x][g]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (j < 2 && i + kAhead < kN1) issue1(i + kAhead, j);
                }
            }
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (r0 < all.lo || r0 + kStepRows > all.hi) {
                auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const int at = r0 + 16 * x + 4 * q4;
                        const unsigned bits = below(mine[g].hi - at) & ~below(mine[g].lo - at);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            s[x][g][i] = (bits >> i) & 1 ? s[x][g][i] : neg_inf();
                            dp[x][g][i] = (bits >> i) & 1 ? dp[x][g][i] : 0.f;
                        }
                    }
            }
            // P and dS, the rows of both blocks the second products' eight
            bf16x8 pb[2], db_[2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                f32x8 a, b;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    a[i] = fast_exp2(s[i >> 2][g][i & 3] * sl2);
                    b[i] = a[i] * dp[i >> 2][g][i & 3];
                }
                pb[g] = __builtin_convertvector(a, bf16x8);
                db_[g] = __builtin_convertvector(b, bf16x8);
            }
            asm volatile("" ::"v"(pb[0]), "v"(pb[1]), "v"(db_[0]), "v"(db_[1]));
            __builtin_amdgcn_sched_barrier(0);
            // dV^T += dO^T P, dK^T += Q^T dS
            constexpr int kN2 = 2 * (kNO / 2), kAhead2 = 3;
            bf16x8 h[kN2][2];
            auto issue2 = [&](int i, int x) { h[i][x] = read_v_frag<D>((i < kNO / 2 ? gt : qt) + (rb.v ^ ((2 * (i % (kNO / 2)) + x) << 5))); };
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < kAhead2; i++) issue2(i, 0), issue2(i, 1);
#pragma unroll
            for (int i = 0; i < kN2; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int x = j >> 1, g = j & 1, db = 2 * (i % (kNO / 2)) + x;
                    __builtin_amdgcn_sched_barrier(0);
                    if (i < kNO / 2) dv[db][g] = mfma16(h[i][x], pb[g], dv[db][g]);
                    else dk[db][g] = mfma16(h[i][x], db_[g], dk[db][g]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (j < 2 && i + kAhead2 < kN2) issue2(i + kAhead2, j);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<0>();
        block_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int key = wkey + 16 * g + i16;
        if (key >= sq.len) continue;
        const size_t dst = ((size_t)(sq.k0 + key) * p.kv_heads + kvh) * D;
        float* part = p.part_dkv + ((size_t)item.share * p.part_keys + (size_t)(kvh * p.key_items.n.by + item.piece) * kRows + (key - key0)) * 2 * D;
#pragma unroll
        for (int db = 0; db < kNO; db++) {
            const int at = 16 * db + 4 * q4;
            f32x4 x = dk[db][g];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] *= p.scale;
            if (split) {
                *reinterpret_cast<f32x4*>(part + at) = x;
                *reinterpret_cast<f32x4*>(part + D + at) = dv[db][g];
            } else if (p.grads_are_bf16) {
                *reinterpret_cast<bf16x4*>((uint16_t*)p.dk + dst + at) = __builtin_convertvector(x, bf16x4);
                *reinterpret_cast<bf16x4*>((uint16_t*)p.dv + dst + at) = __builtin_convertvector(dv[db][g], bf16x4);
            } else {
                *reinterpret_cast<f32x4*>((float*)p.dk + dst + at) = x;
                *reinterpret_cast<f32x4*>((float*)p.dv + dst + at) = dv[db][g];
            }
        }
    }
}

// ---- the queries' gradients ------------------------------------------------------------------------------------------

// 128 rows of one (sequence, key head), 32 a wave, over tiles of 64 keys in LDS, two buffers for K and for V. Q and dO stay in registers; S^T =
// K Q^T and dP^T = V dO^T leave the scores of two rows in a lane, dS the operand of dQ^T += K^T dS, whose K is the
// same tile read across.
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_dq_kernel(const PackedBackParams p) {
    using G = TileGeo<D>;
    constexpr int kNO = D / 16, kNK = D / 32, kTile = G::kTile, kIter = TileDma<4, D>::ITER, kUnits = kIter / 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    lds_u8* smem = (lds_u8*)smem_raw;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q4 = lane >> 4, i16 = lane & 15;
    const PackedItem item = packed_item(p.row_items, blockIdx.x);
    if (item.head < 0) return;
    const int kvh = item.head, group = p.group.by, number = p.row_items.n.by - 1 - item.piece;
    const PagedPiece piece = paged_piece<kRows>(p.row_pieces, p.b, group, number);
    const PackedSeq sq = packed_seq(p.b, piece.seq);
    const int rows = sq.count * group, row0 = piece.tile * kRows;
    if (row0 >= rows) return;
    const PackedWalk w = packed_walk(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group));
    const int e0 = item.share * p.row_chunk, e1 = min(w.n, e0 + p.row_chunk);
    if (item.share > 0 && e0 >= e1) return;
    const bool split = w.n > p.row_chunk;
    const float sl2 = p.sl2;

    const int wrow = row0 + 32 * wave;
    const bool idle = wrow >= rows;
    PagedSight all_see = {0x7fffffff, 0, 0x7fffffff}, mine = {0, 0, 0};
    if (!idle) {
        all_see = packed_all(p.mask, sq, paged_quot(wrow, p.group), paged_quot(min(wrow + 32, rows) - 1, p.group));
        mine = packed_sight(p.mask, sq.pos0 + paged_quot(min(wrow + (lane & 31), rows - 1), p.group), sq.len);
    }
    const PackedWhole whole = packed_whole(w, all_see);
    bf16x8 qf[kNK][2], gf[kNK][2];
    f32x4 s_init[2], d_init[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = wrow + 16 * g + i16, t = paged_quot(r, p.group);
        const long in = (long)(kvh * group + r - t * group) * G::kRow + 16 * q4;
        const uint8_t* q = (const uint8_t*)p.q + (long)(sq.start + t) * p.q_stride + in;
        const uint8_t* go = (const uint8_t*)p.dout + (long)(sq.start + t) * p.dout_stride + in;
#pragma unroll
        for (int dk = 0; dk < kNK; dk++) {
            u32x4 x = {0u, 0u, 0u, 0u}, y = x;
            if (r < rows) x = *reinterpret_cast<const u32x4*>(q + 64 * dk), y = *reinterpret_cast<const u32x4*>(go + 64 * dk);
            qf[dk][g] = __builtin_bit_cast(bf16x8, x);
            gf[dk][g] = __builtin_bit_cast(bf16x8, y);
        }
        f32x2 stat = {0.f, 0.f};
        if (r < rows) stat = p.stats[((long)kvh * p.b.tokens + sq.start) * group + r];
#pragma unroll
        for (int i = 0; i < 4; i++) s_init[g][i] = stat[0], d_init[g][i] = stat[1];
    }
    const TileReadBases rb = both_bases<D>(lane);
    unsigned koff[kIter], voff[kIter];
    packed_offsets<D>(koff, (unsigned)p.k_stride, wave, lane, [](int r) { return both_swz<D>(r); });
    packed_offsets<D>(voff, (unsigned)p.v_stride, wave, lane, [](int r) { return both_swz<D>(r); });
    const uint16_t *kbase = p.k + kvh * D, *vbase = p.v + kvh * D;
    const unsigned slot = (unsigned)(size_t)smem + wave * kIter * 1024;
    auto load = [&](int e, int buf) {
        const int key = w.key(e), left = min(sq.len - key, kTileRows);
        const u32x4 kd = packed_rows(kbase, sq.k0 + key, p.k_stride, left, G::kRow), vd = packed_rows(vbase, sq.k0 + key, p.v_stride, left, G::kRow);
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            packed_issue(kd, koff[2 * u], koff[2 * u + 1], slot + buf * kTile + u * 2048);
            packed_issue(vd, voff[2 * u], voff[2 * u + 1], slot + (2 + buf) * kTile + u * 2048);
        }
    };
    f32x4 dq[kNO][2];
#pragma unroll
    for (int db = 0; db < kNO; db++) dq[db][0] = dq[db][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (e0 < e1) {
        load(e0, 0);
#pragma unroll
        for (int dk = 0; dk < kNK; dk++) asm volatile("" : "+v"(qf[dk][0]), "+v"(qf[dk][1]), "+v"(gf[dk][0]), "+v"(gf[dk][1]));
        asm volatile("" : "+v"(s_init[0]), "+v"(s_init[1]), "+v"(d_init[0]), "+v"(d_init[1]));
        wait_vmcnt<0>();
        block_barrier();
    }
#pragma unroll 1
    for (int e = e0; e < e1; e++) {
        const int buf = (e - e0) & 1;
        if (e + 1 < e1) load(e + 1, buf ^ 1);
        if (!idle) {
            const bool cut = !whole.tile(e);
#pragma unroll
            for (int t = 0; t < 2; t++) {   // 32 keys at a time: the scores of 64 and their operands would not fit the registers
                const lds_u8* kt = smem + buf * kTile + 32 * t * G::kRow;
                const lds_u8* vt = kt + 2 * kTile;
                f32x4 s[2][2], dp[2][2];   // [16 keys][16 rows]
                constexpr int kN1 = 2 * kNK, kAhead = 3;   // groups: d chunk i / 2, K or V; two operands of 16 keys for four products
                bf16x8 f[kN1][2];
                auto issue1 = [&](int i, int x) { f[i][x] = lds_read_b128((i & 1 ? vt : kt) + (rb.k ^ ((i >> 1) << 6)) + x * 16 * G::kRow); };
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int i = 0; i < kAhead; i++) issue1(i, 0), issue1(i, 1);
#pragma unroll
                for (int i = 0; i < kN1; i++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int x = j >> 1, g = j & 1, dk = i >> 1;
                        __builtin_amdgcn_sched_barrier(0);
                        if (i & 1) dp[x][g] = mfma16(f[i][x], gf[dk][g], dk == 0 ? d_init[g] : dp[x][g]);
                        else s[x][g] = mfma16(f[i][x], qf[dk][g], dk == 0 ? s_init[g] : s[x][g]);
                        __builtin_amdgcn_sched_barrier(0);
                        if (j < 2 && i + kAhead < kN1) issue1(i + kAhead, j);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
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
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int g = 0; g < 2; g++) {
                            const int at = w.key(e) + 32 * t + 16 * x + 4 * q4;
                            const unsigned bits = below(both[0][g] - at) | (below(both[2][g] - at) & ~below(both[1][g] - at));
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                s[x][g][i] = (bits >> i) & 1 ? s[x][g][i] : neg_inf();
                                dp[x][g][i] = (bits >> i) & 1 ? dp[x][g][i] : 0.f;
                            }
                        }
                }
                bf16x8 ds[2];
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    f32x8 a;
#pragma unroll
                    for (int i = 0; i < 8; i++) a[i] = fast_exp2(s[i >> 2][g][i & 3] * sl2) * dp[i >> 2][g][i & 3];
                    ds[g] = __builtin_convertvector(a, bf16x8);
                }
                asm volatile("" ::"v"(ds[0]), "v"(ds[1]));
                __builtin_amdgcn_sched_barrier(0);
                constexpr int kAhead2 = kNK < 3 ? kNK : 3;   // groups: d blocks 2 i + {0, 1}
                bf16x8 h[kNK][2];
                auto issue2 = [&](int i, int x) { h[i][x] = read_v_frag<D>(kt + (rb.v ^ ((2 * i + x) << 5))); };
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int i = 0; i < kAhead2; i++) issue2(i, 0), issue2(i, 1);
#pragma unroll
                for (int i = 0; i < kNK; i++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int x = j >> 1, g = j & 1;
                        __builtin_amdgcn_sched_barrier(0);
                        dq[2 * i + x][g] = mfma16(h[i][x], ds[g], dq[2 * i + x][g]);
                        __builtin_amdgcn_sched_barrier(0);
                        if (j < 2 && i + kAhead2 < kNK) issue2(i + kAhead2, j);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<0>();
        block_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = wrow + 16 * g + i16, t = paged_quot(r, p.group);
        if (r >= rows) continue;
        const size_t dst = ((size_t)(sq.start + t) * p.heads + kvh * group + (r - t * group)) * D;
        float* part = p.part_dq + ((size_t)item.share * p.part_rows + (size_t)(kvh * p.row_items.n.by + number) * kRows + (r - row0)) * D;
#pragma unroll
        for (int db = 0; db < kNO; db++) {
            const int at = 16 * db + 4 * q4;
            f32x4 x = dq[db][g];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] *= p.scale;
            if (split) *reinterpret_cast<f32x4*>(part + at) = x;
            else if (p.grads_are_bf16) *reinterpret_cast<bf16x4*>((uint16_t*)p.dq + dst + at) = __builtin_convertvector(x, bf16x4);
            else *reinterpret_cast<f32x4*>((float*)p.dq + dst + at) = x;
        }
    }
}

// The shares of split walks, added in their order: D / 4 threads a row (of dq) or key (twice as many: dk, dv).
template <int D, bool KEYS>
__global__ __launch_bounds__(256) void packed_sum_kernel(const PackedBackParams p) {
    constexpr int kWide = KEYS ? 2 * D : D, kPer = kWide / 4, kSum = 256 / kPer, kPerPiece = kRows / kSum;
    const int c = threadIdx.x % kPer, in = (int)(blockIdx.x % kPerPiece) * kSum + threadIdx.x / kPer, item = blockIdx.x / kPerPiece;
    const PackedItems& items = KEYS ? p.key_items : p.row_items;
    const int kvh = paged_quot(item, items.n), number = item - kvh * items.n.by, group = p.group.by;
    int steps, chunk;
    void* out;
    size_t dst;
    if constexpr (KEYS) {
        const PackedKeys kb = {p.b.k_start, p.b.seqs, p.b.k_tokens};
        const PagedPiece piece = paged_piece<kRows>(p.key_pieces, kb, 1, number);
        const PackedSeq sq = packed_seq(p.b, piece.seq);
        const int key0 = piece.tile * kRows;
        if (key0 + in >= sq.len) return;
        const RowWalk walk = row_walk(p.mask, sq, key0, min(key0 + kRows, sq.len) - 1, group);
        steps = walk.to - walk.from, chunk = p.key_chunk;
        out = 4 * c < D ? p.dk : p.dv;
        dst = ((size_t)(sq.k0 + key0 + in) * p.kv_heads + kvh) * D + 4 * c % D;
    } else {
        const PagedPiece piece = paged_piece<kRows>(p.row_pieces, p.b, group, number);
        const PackedSeq sq = packed_seq(p.b, piece.seq);
        const int rows = sq.count * group, row0 = piece.tile * kRows, r = row0 + in;
        if (r >= rows) return;
        steps = packed_walk(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group)).n, chunk = p.row_chunk;
        const int t = paged_quot(r, p.group);
        out = p.dq;
        dst = ((size_t)(sq.start + t) * p.heads + kvh * group + (r - t * group)) * D + 4 * c;
    }
    if (steps <= chunk) return;   // (one workgroup's, written)
    const int shares = (steps + chunk - 1) / chunk;
    const float* part = (KEYS ? p.part_dkv : p.part_dq) + ((size_t)item * kRows + in) * kWide + 4 * c;
    const size_t next = (size_t)(KEYS ? p.part_keys : p.part_rows) * kWide;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < shares; s++) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(part + s * next);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] += y[i];
    }
    if (p.grads_are_bf16) *reinterpret_cast<bf16x4*>((uint16_t*)out + dst) = __builtin_convertvector(x, bf16x4);
    else *reinterpret_cast<f32x4*>((float*)out + dst) = x;
}

// How a call is cut, and its workspace.
struct BackCut {
    PagedPieces rows, keys;
    size_t row_chunk, row_shares, key_chunk, key_shares;
};
constexpr size_t kMostShares = (size_t)1 << 30;   // bytes of the shares of a kernel: past it its walks are cut less
BackCut back_cut(const PackedCall& c) {
    const size_t group = c.heads / c.kv_heads, units = (size_t)fv_compute_units(), slots = (c.d == 64 ? 3 : 2) * units;
    BackCut cut;
    cut.rows = paged_pieces(kRows, c.seqs, c.tokens, c.max_q, group);
    cut.keys = paged_pieces(kRows, c.seqs, c.k_tokens, c.max_k, 1);
    auto shares_of = [&](const PagedPieces& x, size_t rows, size_t steps, size_t least, size_t bytes) {
        const size_t items = c.kv_heads * (size_t)x.n.by;
        if (items == 0) return (size_t)1;
        const size_t held = x.tiles.by ? items : std::max<size_t>(c.kv_heads * (rows / kRows + 1), items / 2);
        const size_t shares = held < slots ? std::min(slots / held, std::max<size_t>(steps / least, 1)) : 1;
        return std::min(shares, std::max<size_t>(kMostShares / (items * kRows * bytes), 1));
    };
    const size_t key_steps = fv_packed_key_steps(c, kRows), rows = c.max_q * group;
    size_t row_steps = (rows + kStepRows - 1) / kStepRows;
    if (c.causal && c.window > 0 && c.sink == 0) {   // rows of the window's blocks and of those of the piece's keys
        const size_t blocks = c.window + (kRows + c.block_tokens - 1) / c.block_tokens, far = (size_t)1 << 31;
        const size_t band = blocks < far / c.block_tokens / group ? blocks * c.block_tokens * group : far;
        row_steps = std::min(row_steps, (band + kStepRows - 1) / kStepRows + 1);
    }
    row_steps = std::max<size_t>(row_steps, 1);
    size_t n = shares_of(cut.rows, c.tokens * group, key_steps, 4, c.d * 4);
    cut.row_chunk = (key_steps + n - 1) / n, cut.row_shares = (key_steps + cut.row_chunk - 1) / cut.row_chunk;
    n = shares_of(cut.keys, c.k_tokens, row_steps, 8, c.d * 8);
    cut.key_chunk = (row_steps + n - 1) / n, cut.key_shares = (row_steps + cut.key_chunk - 1) / cut.key_chunk;
    return cut;
}
struct BackParts {
    size_t stats = 0, rounded = 0, dq = 0, dkv = 0, bytes = 0;   // bytes from the workspace's start
    size_t rows, keys;
    BackParts(const PackedCall& c, const BackCut& cut, bool round) {
        auto take = [this](size_t n) {
            const size_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        rows = c.kv_heads * (size_t)cut.rows.n.by * kRows, keys = c.kv_heads * (size_t)cut.keys.n.by * kRows;
        stats = take(c.tokens * c.heads * 8);
        if (round) rounded = take(c.tokens * c.heads * c.d * 2);
        if (cut.row_shares > 1) dq = take(cut.row_shares * rows * c.d * 4);
        if (cut.key_shares > 1) dkv = take(cut.key_shares * keys * c.d * 8);
    }
};
constexpr int dkv_lds(int d) { return kRows * d * 2 + 4 * kStepRows * d * 2 + 2 * 256; }
std::atomic<unsigned long long> lds_done{0};

}  // namespace
}  // namespace fv

extern "C" {

size_t fv_packed_attention_backward_workspace_bytes(int dout_is_bf16, size_t heads, size_t kv_heads, size_t d, size_t seqs, size_t q_tokens,
                                                    size_t k_tokens, size_t max_q, size_t max_k, int causal, size_t block_tokens, size_t window,
                                                    size_t sink) {
    const PackedCall c = {heads, kv_heads, d, seqs, q_tokens, k_tokens, std::min(max_q, q_tokens), std::min(max_k, k_tokens), nullptr, nullptr, 1.f, causal,
                          block_tokens, window, sink};
    return fv_packed_sizes(c) ? fv::BackParts(c, fv::back_cut(c), !dout_is_bf16).bytes : 0;
}

int fv_packed_attention_backward(const void* dout, int dout_is_bf16, const uint16_t* q, size_t q_stride, const uint16_t* k, size_t k_stride,
                                 const uint16_t* v, size_t v_stride, const void* out, int out_is_bf16, const float* lse, void* dq, void* dk, void* dv,
                                 int grads_are_bf16, size_t heads, size_t kv_heads, size_t d, const int32_t* q_start, const int32_t* k_start,
                                 size_t seqs, size_t q_tokens, size_t k_tokens, size_t max_q, size_t max_k, float scale, int causal,
                                 size_t block_tokens, size_t window, size_t sink, void* workspace, size_t workspace_bytes, void* stream) {
    if (seqs == 0 || (q_tokens == 0 && k_tokens == 0)) return FV_OK;   // (empty arrays may have no address)
    const PackedCall c = {heads, kv_heads, d, seqs, q_tokens, k_tokens, std::min(max_q, q_tokens), std::min(max_k, k_tokens), q_start, k_start, scale,
                          causal, block_tokens, window, sink};
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
    const fv::BackCut cut = fv::back_cut(c);
    const fv::BackParts parts(c, cut, !dout_is_bf16);
    if (parts.bytes > 0 && (!workspace || workspace_bytes < parts.bytes)) return fv_invalid("packed attention backward: workspace too small");
    const size_t row_items = kv_heads * (size_t)cut.rows.n.by, key_items = kv_heads * (size_t)cut.keys.n.by;
    const size_t rows = q_tokens * heads, stat_blocks = (rows + 2048 / d - 1) / (2048 / d);
    const size_t sum_rows = row_items * fv::kRows / (1024 / d), sum_keys = key_items * fv::kRows / (512 / d);
    constexpr size_t kMost = (size_t)1 << 24;   // (a launch holds fewer than 2^32 work-items)
    if (row_items * cut.row_shares >= kMost / 2 || key_items * cut.key_shares >= kMost / 2 || stat_blocks >= kMost ||
        (cut.row_shares > 1 && sum_rows >= kMost) || (cut.key_shares > 1 && sum_keys >= kMost))
        return fv_decline("packed attention backward: too large for one launch");
    uint8_t* ws = (uint8_t*)workspace;
    fv::PackedBackParams p;
    p.b = {q_start, k_start, (int)seqs, (int)q_tokens, (int)k_tokens, (int)c.max_q, (int)c.max_k};
    p.mask = fv_packed_mask(c);
    p.q = q, p.k = k, p.v = v, p.dout = dout_is_bf16 ? (const uint16_t*)dout : (const uint16_t*)(ws + parts.rounded);
    p.q_stride = (long)q_stride * 2, p.k_stride = (long)k_stride * 2, p.v_stride = (long)v_stride * 2, p.dout_stride = (long)(heads * d * 2);
    p.stats = (const fv::f32x2*)(ws + parts.stats);
    p.dq = dq, p.dk = dk, p.dv = dv, p.grads_are_bf16 = grads_are_bf16 != 0;
    p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = fv::paged_div(heads / kv_heads);
    p.scale = scale, p.sl2 = (float)((double)scale * 1.4426950408889634);
    p.row_pieces = cut.rows, p.key_pieces = cut.keys;
    p.row_items = fv::packed_items(kv_heads, (size_t)cut.rows.n.by, cut.row_shares);
    p.key_items = fv::packed_items(kv_heads, (size_t)cut.keys.n.by, cut.key_shares);
    p.row_chunk = (int)cut.row_chunk, p.key_chunk = (int)cut.key_chunk;
    p.part_dq = (float*)(ws + parts.dq), p.part_dkv = (float*)(ws + parts.dkv), p.part_rows = (long)parts.rows, p.part_keys = (long)parts.keys;
    hipStream_t st = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    fv::paged_pick(d == 128, [&](auto d128) {
        constexpr int D = d128() ? 128 : 64;
        if (D == 128) e = fv_set_max_lds_once((const void*)fv::packed_dkv_kernel<D>, fv::dkv_lds(D), fv::lds_done);
        if (e != hipSuccess) return;
        if (q_tokens > 0)
            fv::paged_pick(out_is_bf16 != 0, [&](auto o16) {
                fv::paged_pick(dout_is_bf16 != 0, [&](auto g16) {
                    hipLaunchKernelGGL((fv::packed_stats_kernel<D, o16(), g16()>), dim3((unsigned)stat_blocks), dim3(256), 0, st, dout, out, lse,
                                       (fv::f32x2*)(ws + parts.stats), (uint16_t*)(ws + parts.rounded), (long)rows, (long)q_tokens, (int)heads, p.group,
                                       (float)(1.0 / (double)scale));
                });
            });
        if (key_items > 0) {
            hipLaunchKernelGGL((fv::packed_dkv_kernel<D>), dim3((unsigned)fv::packed_blocks(p.key_items)), dim3(256), fv::dkv_lds(D), st, p);
            if (cut.key_shares > 1) hipLaunchKernelGGL((fv::packed_sum_kernel<D, true>), dim3((unsigned)sum_keys), dim3(256), 0, st, p);
        }
        if (row_items > 0) {
            hipLaunchKernelGGL((fv::packed_dq_kernel<D>), dim3((unsigned)fv::packed_blocks(p.row_items)), dim3(256), 4 * fv::TileGeo<D>::kTile, st, p);
            if (cut.row_shares > 1) hipLaunchKernelGGL((fv::packed_sum_kernel<D, false>), dim3((unsigned)sum_rows), dim3(256), 0, st, p);
        }
    });
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "packed_attention_backward");
}

}  // extern "C"
