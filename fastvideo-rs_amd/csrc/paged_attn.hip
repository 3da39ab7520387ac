// Attention over a paged KV cache (declarations: include/fv_sdpa_hip.h): for every row (token t of a sequence, query head h)
// at position p, o = sum_j softmax_j(scale q . k_j) v_j over the keys j that it sees: block(j) <= block(p), and within the
// window of blocks or among the sink blocks.
//
// Rows of one key head lie together (token by token, the heads of its group in turn), so a step over 32 keys serves all of
// them with one load of K and V. Scores, offsets, sums and O are f32; the probabilities are rounded to bf16 for the second product (each
// off by 2^-8 of itself at most, as much as a result in bf16 is), 4-bit keys and values become bf16 exactly.
#include <limits.h>

#include <algorithm>

#include "../../include/fv_sdpa_hip.h"
#include "attn_core.h"
#include "fv_common.h"
#include "fv_internal.h"
#include "paged.h"

namespace fv {
namespace {

constexpr int kStep = 32;       // keys a wave takes at a time
constexpr int kWaves = 4;
constexpr float kLeast = 0x1p-149f;   // the weight of a seen key that vanished, where its value is not finite

struct PagedAttnParams {
    PagedPool pool;
    PagedBatch b;
    const uint16_t* q;
    long q_stride;              // elements between tokens
    void* out;                  // [tokens, heads, d]
    int out_is_bf16;
    int heads;
    PagedDiv group;             // query heads that share a key head
    float sl2;                  // scale * log2(e)
    PagedDiv block_tokens;
    int window, sink;           // blocks; window 0: all
    // Two kernels share a call: sequences of up to `few` rows a key head go to paged_rows_kernel, the others to
    // paged_tiles_kernel. How each cuts its part:
    int few;
    int rows_m;                 // rows a tile of paged_rows_kernel
    PagedDiv rows_tiles, kv_heads;   // (tiles of a (sequence, key head) there)
    PagedDiv rows_chunk, rows_chunks;   // steps of the walk that a workgroup takes, workgroups a walk
    PagedDiv big_chunk;         // (steps)
    // paged_tiles_kernel: the first big_full tiles (a multiple of 8), counted key head by key head and the last rows first, have a
    // workgroup each, the others as many as they have shares: big_rest workgroups, in sets of big_set tiles and big_set_shares shares.
    PagedPieces big_pieces;
    int big_full, big_rest;
    PagedDiv big_set, big_set_shares;
    int xcds;                   // 2^xcds XCDs share a run of items
    // Shares: values, each normalised, and the base-2 logarithm of its sum. Of paged_rows_kernel [chunks][`few` rows of each (sequence, key head)][d] and
    // [chunks][these rows], of paged_tiles_kernel [chunks][128 rows of each tile that is cut] likewise.
    float *rows_o, *rows_lse, *big_o, *big_lse;
    long big_rows;              // the latter's rows
    // paged_join_kernel: the first join_tiles workgroups those of the cut tiles, then join_few each of a (sequence, key head) of few rows
    int join_tiles;
    PagedDiv join_few;
};

// The walk of a tile of rows (tokens t0 .. t1 of the sequence) in steps of STEP keys: [0, ns) hold the sink, then
// [b0, b0 + n - ns).
template <int STEP>
struct PagedWalk {
    int ns, b0, n;
    PagedSight any;             // the keys that some row sees
    FV_DEV int key(int e) const { return (e < ns ? e : b0 + e - ns) * STEP; }
};
// Whether rows all of which see `all` see every key of [k, e).
FV_DEV bool paged_whole(const PagedSight& all, int k, int e) {
    return e <= all.a || (k >= all.lo && e <= all.hi) || (all.a >= all.lo && e <= all.hi);
}
template <class Params>
FV_DEV PagedSight paged_all(const Params& p, const PagedSeq& s, int t0, int t1) {   // what the tokens t0 .. t1 all see
    const PagedSight f = paged_sight(p, s.first_pos() + t0, s.len), l = paged_sight(p, s.first_pos() + t1, s.len);
    return {f.a, l.lo, f.hi};
}
template <int STEP, class Params>
FV_DEV PagedWalk<STEP> paged_walk(const Params& p, const PagedSeq& s, int t0, int t1) {
    PagedWalk<STEP> w;
    const PagedSight l = paged_sight(p, s.first_pos() + t1, s.len);
    w.any = {l.a, paged_sight(p, max(s.first_pos() + t0, 0), s.len).lo, l.hi};
    w.ns = (w.any.a + STEP - 1) / STEP;
    w.b0 = max(w.any.lo / STEP, w.ns);
    w.n = w.ns + max(0, (w.any.hi + STEP - 1) / STEP - w.b0);
    return w;
}

// What a lane holds of one step: lane l takes part in the products as row l % 16 and K group l / 16.
//   K: its rows of two blocks of 16 keys. Row r of block b is key 8 (r / 4) + 4 b + r % 4, so that the scores S = K Q^T, whose
//      lane has rows 4 (l / 16) .. + 3 of both blocks, are those of keys 8 (l / 16) .. + 7 in order: the probabilities are
//      the operand of the second product as they stand.
//   V: 8 keys, 8 (l / 16) .. + 7, of D / 16 channels, (D / 16) (l % 16) .. : turned over within the lane (v_perm_b32) they are the
//      operands V^T of D / 16 products, channel (D / 16) r + c in row r of the c-th. Nothing passes through LDS.
template <int D, bool FOUR>
struct PagedStage;
template <int D>
struct PagedStage<D, false> {
    static constexpr int kWords = D / 32;                  // words of D / 16 channels
    typedef __attribute__((ext_vector_type(kWords))) unsigned vwords;
    u32x4 k[2][D / 32];
    vwords v[8];
};
template <int D>
struct PagedStage<D, true> {
    static constexpr int kWords = D / 32;
    typedef __attribute__((ext_vector_type(D / 32))) unsigned kwords;   // D / 4 codes of a key
    kwords k[2];
    unsigned kscale[2];
    unsigned v[8];                                          // D / 16 codes of a key (D = 64: in the low half)
    u32x4 vscale[D / 64];                                   // the scales of the lane's 8 keys
};

template <int D, bool FOUR>
struct PagedLane {
    const uint8_t *k, *v, *ks, *vs;    // the lane's place in a half step of 16 keys at the pool's first row
};

template <int D, bool FOUR>
FV_DEV void paged_load_k(PagedStage<D, FOUR>& s, const PagedLane<D, FOUR>& at, unsigned row0, unsigned row1, int lane) {
    constexpr int kRow = PagedGeo<D, FOUR>::kRow;
    const size_t row = (lane & 8) ? row1 : row0;
    const uint8_t* k = at.k + row * kRow;
    if constexpr (FOUR) {
        constexpr int kS = PagedGeo<D, true>::kScales;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            s.k[b] = *reinterpret_cast<const typename PagedStage<D, true>::kwords*>(k + 4 * b * kRow);
            s.kscale[b] = at.ks[row * kS + 4 * b * kS];
        }
    } else {
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int dk = 0; dk < D / 32; dk++) s.k[b][dk] = *reinterpret_cast<const u32x4*>(k + 4 * b * kRow + 64 * dk);
    }
}
template <int D, bool FOUR>
FV_DEV void paged_load_v(PagedStage<D, FOUR>& s, const PagedLane<D, FOUR>& at, unsigned row0, unsigned row1, int lane) {
    constexpr int kRow = PagedGeo<D, FOUR>::kRow;
    const size_t row = (lane & 32) ? row1 : row0;
    const uint8_t* v = at.v + row * kRow;
    if constexpr (FOUR) {
        constexpr int kS = PagedGeo<D, true>::kScales;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (D == 128) s.v[j] = *reinterpret_cast<const unsigned*>(v + j * kRow);
            else s.v[j] = *reinterpret_cast<const uint16_t*>(v + j * kRow);
        }
#pragma unroll
        for (int j = 0; j < D / 64; j++) s.vscale[j] = *reinterpret_cast<const u32x4*>(at.vs + row * kS + 16 * j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) s.v[j] = *reinterpret_cast<const typename PagedStage<D, false>::vwords*>(v + j * kRow);
    }
}

template <int D, bool FOUR>
FV_DEV void paged_lane(PagedLane<D, FOUR>& at, const PagedPool& pool, int lane) {
    constexpr int kRow = PagedGeo<D, FOUR>::kRow, kS = PagedGeo<D, FOUR>::kScales;
    const int r = lane & 15, g = lane >> 4;
    const int krow = 8 * ((r >> 2) & 1) + (r & 3), vrow = 8 * (g & 1);
    at.k = (const uint8_t*)pool.k + krow * kRow + (FOUR ? g * (D / 8) : 16 * g);
    at.v = (const uint8_t*)pool.v + vrow * kRow + r * (kRow / 16);
    if constexpr (FOUR) {
        at.ks = pool.ks + krow * kS + g * kS / 4;
        at.vs = pool.vs + vrow * kS;
    } else {
        at.ks = at.vs = nullptr;
    }
}

// The K operand of block b, piece dk: channels 32 dk + 8 g .. + 7 of a bf16 key, (D / 4) g + 8 dk .. + 7 of a 4-bit one.
template <int D, bool FOUR>
FV_DEV bf16x8 k_frag(const PagedStage<D, FOUR>& s, int b, int dk) {
    if constexpr (FOUR) return __builtin_bit_cast(bf16x8, fp4_eight(s.k[b][dk], e8m0_scale(s.kscale[b])));
    else return __builtin_bit_cast(bf16x8, s.k[b][dk]);
}
// Word X of the lane's V as bf16, channels 2 X and 2 X + 1 of its D / 16, of each of its 8 keys.
template <int D, bool FOUR>
struct VScales {
    float of[FOUR ? 8 : 1];
    FV_DEV VScales(const PagedStage<D, FOUR>& s, int lane) {
        if constexpr (FOUR) {
            constexpr int kS = D / 32;                        // scale bytes a key
            const int shift = 8 * ((lane & 15) * (D / 16) / 32);
#pragma unroll
            for (int j = 0; j < 8; j++) of[j] = e8m0_scale((s.vscale[j * kS / 16][(j * kS / 4) & 3] >> (shift + 8 * (j * kS & 3))) & 255u);
        }
    }
};
template <int X, int D, bool FOUR>
FV_DEV void v_words(const PagedStage<D, FOUR>& s, const VScales<D, FOUR>& scales, unsigned (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if constexpr (FOUR) w[j] = fp4_pair<X>(s.v[j], scales.of[j]);
        else w[j] = s.v[j][X];
    }
}

// N channels from `c` of row `row` of the values as they stand in the pool.
template <int D, bool FOUR, int N, class Pool>
FV_DEV void pool_values(const Pool& pool, unsigned row, int c, float (&v)[N]) {
    if constexpr (FOUR) {
        const uint8_t* at = (const uint8_t*)pool.v + (size_t)row * (D / 2) + c / 2;
        const float scale = e8m0_scale(pool.vs[(size_t)row * (D / 32) + c / 32]);   // (N channels lie in one block)
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const unsigned w = fp4_pair<0>(at[i / 2], scale);
            v[i] = __builtin_bit_cast(float, w << 16);
            v[i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
        }
    } else {
        const uint16_t* at = (const uint16_t*)pool.v + (size_t)row * D + c;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = bf16_bits_to_f32(at[i]);
    }
}

// One workgroup: a share of the walk of a tile of 16 NT rows of one (sequence, key head); its four waves take the share's
// steps in turn, each with a running maximum of its own, and join through LDS. A step reads its keys and values once, for all of
// the tile's rows, straight into registers in the order of the matrix operands, so that nothing but the memory bounds it: 64
// single tokens of 40 / 8 heads over 1.24 GB of bf16 pages 237 us, 5.2 TB/s; 40 such over 0.85 GB of 4 bits 173 us, 4.9. Calls too
// short for that are bound by their few waits in a row: 4 tokens of 24 heads over up to 777 keys of 64 channels 9.2 us.
// One tile of rows: a whole step is loaded ahead. Two (4-bit pages, few_rows): the keys of the next step go into the registers of
// this one's as soon as their scores are there, its values likewise; a whole step ahead spilled 270 bytes a lane.
template <int D, bool FOUR, int NT>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(const PagedAttnParams p) {
    constexpr int kNO = D / 16, kPad = D + 4, kDepth = NT == 1 ? 2 : 1;
    __shared__ float lds_o[kWaves][16][kPad];
    __shared__ float lds_ml[kWaves][16][2], lds_row[16][2];   // a wave's (offset, sum) of its rows; (1 / sum, log2 of the sum) of all
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    int item = blockIdx.x;
    auto digit = [&](const PagedDiv& d) {   // of the workgroup's number, the last one
        const int q = paged_quot(item, d), r = item - q * d.by;
        item = q;
        return r;
    };
    const int tile = digit(p.rows_tiles), kvh = digit(p.kv_heads), chunk = digit(p.rows_chunks), seq = item;
    const PagedSeq sq = paged_seq(p.b, seq);
    const int rows = sq.count * p.group.by, row0 = tile * 16 * NT;
    if (row0 >= rows || rows > p.few) return;
    const int t0 = paged_quot(row0, p.group), t1 = paged_quot(min(row0 + 16 * NT, rows) - 1, p.group);
    const PagedWalk<kStep> w = paged_walk<kStep>(p, sq, t0, t1);
    const PagedSight all_see = paged_all(p, sq, t0, t1);
    const int e0 = chunk * p.rows_chunk.by, e1 = min(w.n, e0 + p.rows_chunk.by);
    if (chunk > 0 && e0 >= e1) return;

    PagedSight see[NT];
    bf16x8 qf[NT][D / 32];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = row0 + 16 * n + col, t = paged_quot(r, p.group), h = kvh * p.group.by + r - t * p.group.by;
        const bool ok = r < rows;
        see[n] = paged_sight(p, ok ? sq.first_pos() + t : -1, sq.len);
        const uint16_t* q = p.q + (size_t)(sq.start + t) * p.q_stride + h * D + (FOUR ? (D / 4) * g : 8 * g);
#pragma unroll
        for (int dk = 0; dk < D / 32; dk++) {
            u32x4 x = {0u, 0u, 0u, 0u};
            if (ok) x = *reinterpret_cast<const u32x4*>(q + (FOUR ? 8 : 32) * dk);
            qf[n][dk] = __builtin_bit_cast(bf16x8, x);
        }
    }
    f32x4 o[NT][kNO];
    float off[NT], l[NT];       // the offset of the lane's row in raw scores, the lane's share of its sum
    bool some[NT];              // whether the row has seen a score (its offset is set)
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int c = 0; c < kNO; c++) o[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        off[n] = l[n] = 0.f;
        some[n] = false;
    }
    PagedLane<D, FOUR> at;
    paged_lane<D, FOUR>(at, p.pool, lane);
    const int* table = p.b.table + (size_t)seq * p.b.table_stride;
    const int lg = p.pool.lg, slots = (1 << lg) - 1, columns = (p.b.max_len + slots) >> lg;

    // S = K Q^T of a step, relative to the rows' offsets
    auto scores = [&](const PagedStage<D, FOUR>& s, f32x4 (&x)[NT][2]) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float m = -off[n];
            x[n][0] = x[n][1] = f32x4{m, m, m, m};
        }
#pragma unroll
        for (int dk = 0; dk < D / 32; dk++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const bf16x8 kf = k_frag<D, FOUR>(s, b, dk);
#pragma unroll
                for (int n = 0; n < NT; n++) x[n][b] = mfma16(kf, qf[n][dk], x[n][b]);
            }
    };
    auto softmax = [&](f32x4 (&x)[NT][2], bf16x8 (&pr)[NT], int k0, unsigned good) {
        const int kl = k0 + 8 * g;
        if (!paged_whole(all_see, k0, k0 + kStep) || good != 3) {   // keys that a row does not see, keys of pages that are none
            const unsigned mask = (good >> (g >> 1)) & 1 ? 0xffu : 0u;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const unsigned seen = see[n].eight(kl) & mask;
#pragma unroll
                for (int j = 0; j < 8; j++) x[n][j >> 2][j & 3] = (seen >> j) & 1 ? x[n][j >> 2][j & 3] : neg_inf();
            }
        }
        bool need = false;
        float mx[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float m = x[n][0][0];
#pragma unroll
            for (int j = 1; j < 8; j++) m = __builtin_fmaxf(m, x[n][j >> 2][j & 3]);
            mx[n] = quad_max(m);
            need |= mx[n] * p.sl2 > 6.0f || (!some[n] && mx[n] > neg_inf());
        }
        if (__builtin_amdgcn_ballot_w64(need) != 0) {   // rare: a row's maximum has outgrown its offset by 2^6, or is its first
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const bool move = mx[n] > neg_inf() && (!some[n] || mx[n] > 0.f);
                const float delta = move ? mx[n] : 0.f;
                const float alpha = some[n] ? fast_exp2(-delta * p.sl2) : 0.f;
                l[n] *= alpha;
                off[n] += delta;
                some[n] |= mx[n] > neg_inf();
#pragma unroll
                for (int c = 0; c < kNO; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[n][c][i] *= alpha;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[n][b][i] -= delta;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            f32x8 e;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = fast_exp2(x[n][j >> 2][j & 3] * p.sl2);
                l[n] += e[j];
            }
            pr[n] = __builtin_convertvector(e, bf16x8);   // (the second product's operand; the sum keeps all of f32)
        }
    };
    auto add_values = [&](const PagedStage<D, FOUR>& s, const bf16x8 (&pr)[NT], int k0, unsigned good, unsigned row_a, unsigned row_b) {
        const VScales<D, FOUR> scales(s, lane);
        const bool whole = paged_whole(all_see, k0, k0 + kStep) && good == 3;
        // values that no row sees are zeros, whatever they are
        unsigned used = whole ? 0xffu : w.any.eight(k0 + 8 * g) & ((good >> (g >> 1)) & 1 ? 0xffu : 0u);
        if (!whole && t0 != t1) {
            // A value that is not finite belongs to the rows that see it, whatever its weight: a probability of zero does not keep it
            // from the others. Its key leaves the product, and the rows that see it add their shares one by one. (Rare.)
            float bad[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            auto look = [&](auto x) {
                unsigned vw[8];
                v_words<x()>(s, scales, vw);
#pragma unroll
                for (int j = 0; j < 8; j++) bad[j] = not_finite(vw[j], bad[j]);
            };
            look(std::integral_constant<int, 0>{});
            look(std::integral_constant<int, 1>{});
            if constexpr (D == 128) {
                look(std::integral_constant<int, 2>{});
                look(std::integral_constant<int, 3>{});
            }
            unsigned out_of_it = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) out_of_it |= bad[j] != 0.f ? 1u << j : 0u;
            out_of_it &= used;
            if (__builtin_amdgcn_ballot_w64(out_of_it != 0) != 0) {
#pragma unroll 1
                for (int x = 0; x < 32; x++) {   // key x of the step: bit x % 8 of lanes 16 (x / 8) ..
                    const int j = x & 7, h = x >> 3;
                    if (((__builtin_amdgcn_ballot_w64((out_of_it >> j) & 1) >> (16 * h)) & 0xffff) == 0) continue;
                    if (g == h) out_of_it |= 1u << j;   // (of all lanes that hold the key)
                    const unsigned row = (h < 2 ? row_a : row_b) + 8 * (h & 1) + j;
                    float pj[NT];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const u32x4 all = __builtin_bit_cast(u32x4, pr[n]);
                        const unsigned pair = j < 4 ? (j < 2 ? all[0] : all[1]) : (j < 6 ? all[2] : all[3]);
                        pj[n] = __shfl(__builtin_bit_cast(float, j & 1 ? pair & 0xffff0000u : pair << 16), 16 * h + col, 64);
                        if (pj[n] == 0.f && see[n].one(k0 + x)) pj[n] = kLeast;
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float v[kNO];
                        pool_values<D, FOUR>(p.pool, row, (D / 4) * g + kNO * i, v);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int c = 0; c < kNO; c++) o[n][c][i] += pj[n] == 0.f ? 0.f : pj[n] * v[c];
                    }
                }
            }
            used &= ~out_of_it;
        }
        auto word = [&](auto x) {
            unsigned vw[8];
            v_words<x()>(s, scales, vw);
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8; j++) vw[j] = (used >> j) & 1 ? vw[j] : 0u;
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                u32x4 t;
#pragma unroll
                for (int i = 0; i < 4; i++) t[i] = __builtin_amdgcn_perm(vw[2 * i + 1], vw[2 * i], c ? 0x07060302u : 0x05040100u);
                const bf16x8 vf = __builtin_bit_cast(bf16x8, t);
#pragma unroll
                for (int n = 0; n < NT; n++) o[n][2 * x() + c] = mfma16(vf, pr[n], o[n][2 * x() + c]);
            }
        };
        word(std::integral_constant<int, 0>{});
        word(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
            word(std::integral_constant<int, 2>{});
            word(std::integral_constant<int, 3>{});
        }
    };

    // groups of 64 steps of the wave: their page numbers are fetched at once, one a lane
    for (int first = e0 + wave; first < e1; first += 64 * kWaves) {
        const int mine = first + lane * kWaves;
        const int my_key = w.key(min(mine, e1 - 1));
        const int my_page = my_key >> lg;
        const int id0 = table[my_page];
        const int id1 = lg == 4 ? table[min(my_page + 1, columns - 1)] : id0;
        const int count = min(64, (e1 - first + kWaves - 1) / kWaves);
        struct Step {
            int key;
            unsigned row[2], good;   // of its halves of 16 keys: first row in the pool, whether the page is one of the pool's
        };
        auto step = [&](int i) {     // (past the group's end: its last step again)
            i = min(i, count - 1);
            const int a = __builtin_amdgcn_readlane(id0, i), b = __builtin_amdgcn_readlane(id1, i);
            Step x;
            x.key = w.key(first + i * kWaves);
            const bool ga = (unsigned)a < (unsigned)p.pool.pages, gb = (unsigned)b < (unsigned)p.pool.pages;
            x.good = (ga ? 1u : 0u) | (gb ? 2u : 0u);
            x.row[0] = (((unsigned)(ga ? a : 0) * (unsigned)p.pool.kv_heads + (unsigned)kvh) << lg) + (unsigned)(x.key & slots);
            x.row[1] = lg == 4 ? ((unsigned)(gb ? b : 0) * (unsigned)p.pool.kv_heads + (unsigned)kvh) << lg : x.row[0] + 16;
            return x;
        };
        PagedStage<D, FOUR> stage[kDepth];
        Step now = step(0);
        paged_load_k<D, FOUR>(stage[0], at, now.row[0], now.row[1], lane);
        paged_load_v<D, FOUR>(stage[0], at, now.row[0], now.row[1], lane);
        for (int i = 0; i < count; i += kDepth) {
#pragma unroll
            for (int x = 0; x < kDepth; x++) {
                if (i + x >= count) break;
                PagedStage<D, FOUR>&s = stage[x], &ahead = stage[kDepth - 1 - x];
                const Step next = step(i + x + 1);
                f32x4 sc[NT][2];
                bf16x8 pr[NT];
                if constexpr (kDepth > 1) {
                    paged_load_k<D, FOUR>(ahead, at, next.row[0], next.row[1], lane);
                    paged_load_v<D, FOUR>(ahead, at, next.row[0], next.row[1], lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                scores(s, sc);
                if constexpr (kDepth == 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    paged_load_k<D, FOUR>(s, at, next.row[0], next.row[1], lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                softmax(sc, pr, now.key, now.good);
                add_values(s, pr, now.key, now.good, now.row[0], now.row[1]);
                if constexpr (kDepth == 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    paged_load_v<D, FOUR>(s, at, next.row[0], next.row[1], lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                now = next;
            }
        }
    }

    // join the waves: each brings its rows' offsets and sums, and its O scaled to the common offset
    const bool split = w.n > p.rows_chunk.by;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float sum = quad_sum(l[n]);
        const float m2 = some[n] ? off[n] * p.sl2 : neg_inf();
        if (g == 0) lds_ml[wave][col][0] = m2, lds_ml[wave][col][1] = sum;
        __syncthreads();
        float top = neg_inf(), total = 0.f;
#pragma unroll
        for (int x = 0; x < kWaves; x++) top = __builtin_fmaxf(top, lds_ml[x][col][0]);
#pragma unroll
        for (int x = 0; x < kWaves; x++) {
            const float mx = lds_ml[x][col][0];
            total += mx == neg_inf() ? lds_ml[x][col][1] : lds_ml[x][col][1] * fast_exp2(mx - top);
        }
        const float scale = m2 == neg_inf() ? 1.f : fast_exp2(m2 - top);
        // lane: channels (D / 4) g + kNO i + c of its row
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < kNO; c += 4)
                *reinterpret_cast<f32x4*>(&lds_o[wave][col][(D / 4) * g + kNO * i + c]) =
                    f32x4{o[n][c][i] * scale, o[n][c + 1][i] * scale, o[n][c + 2][i] * scale, o[n][c + 3][i] * scale};
        const float inv = total == 0.f ? 0.f : 1.f / total;
        if (wave == 0 && g == 0) lds_row[col][0] = inv, lds_row[col][1] = top == neg_inf() ? (total == 0.f ? neg_inf() : total) : top + __log2f(total);
        __syncthreads();
        {
            constexpr int kPer = D / 16;   // channels a thread stores
            const int rr = threadIdx.x >> 4, cc = (threadIdx.x & 15) * kPer;
            const int r = row0 + 16 * n + rr;
            if (r < rows) {
                const int t = paged_quot(r, p.group);
                const size_t dst = (size_t)(sq.start + t) * p.heads + kvh * p.group.by + (r - t * p.group.by);
                const float k = lds_row[rr][0];
                float val[kPer];
#pragma unroll
                for (int c = 0; c < kPer; c++) {
                    float a = 0.f;
#pragma unroll
                    for (int x = 0; x < kWaves; x++) a += lds_o[x][rr][cc + c];
                    val[c] = a * k;
                }
                if (split) {
                    const size_t share = ((size_t)chunk * p.b.seqs * p.kv_heads.by + (size_t)seq * p.kv_heads.by + kvh) * p.few + r;
                    float* po = p.rows_o + share * D + cc;
#pragma unroll
                    for (int c = 0; c < kPer; c += 4) *reinterpret_cast<f32x4*>(po + c) = f32x4{val[c], val[c + 1], val[c + 2], val[c + 3]};
                    if (cc == 0) p.rows_lse[share] = lds_row[rr][1];
                } else if (p.out_is_bf16) {
                    __attribute__((ext_vector_type(kPer))) float f;
#pragma unroll
                    for (int c = 0; c < kPer; c++) f[c] = val[c];
                    typedef __attribute__((ext_vector_type(kPer))) __bf16 bfv;
                    *reinterpret_cast<bfv*>((uint16_t*)p.out + dst * D + cc) = __builtin_convertvector(f, bfv);
                } else {
#pragma unroll
                    for (int c = 0; c < kPer; c += 4)
                        *reinterpret_cast<f32x4*>((float*)p.out + dst * D + cc + c) = f32x4{val[c], val[c + 1], val[c + 2], val[c + 3]};
                }
            }
        }
        if (NT > 1) __syncthreads();
    }
}

// Sequences of many rows: a workgroup takes 128 rows of one (sequence, key head), 32 a wave, over tiles of 64 keys that pass
// through LDS as in the dense kernels (attn_core.h): two buffers for K, two for V. A phase is one key tile: the matrix part
// (O += P V of the tile before, S = K Q^T) with the next K and this V on their way in, the softmax, one barrier. A wave brings
// 16 keys of each tile, which lie in one page whatever its size, so a page costs a tile one lookup; a tile is any four parts of 16 in
// the walk's order, so a few sink tokens and a window that begins anywhere cost no tile of their own (prompts of up to 6001 tokens, 32 / 8
// heads, a window of 1024 with 4 sinks: 227 us; in tiles of 64 neighbouring keys 240):
//   bf16 pages: loads straight to LDS through a buffer descriptor of the wave's 16 rows, whose length cuts off what lies
//     behind the sequence's last key (zeros in LDS, whatever the page holds);
//   4-bit pages: a lane has a quarter of a row in registers a phase ahead and writes it to LDS as bf16 between the matrix
//     instructions, 4 conversions and a write at a time.
constexpr int kBigRows = 128, kPart = 16;   // keys that a wave brings of a tile
// The softmax's vector work, about two thirds of a phase's matrix time, and the matrix work bound it together, and only in part
// overlap between a unit's two workgroups: one frame of 1560 rows x 12 heads against 32760 293 us, 1.07 PFLOP/s of the large product's
// 1.35, the matrix cores busy 60 % of the time while all units have work; three frames of two sequences over 4 bits 1.51 ms, 1.25. (Tried and slower: 8 waves in
// two groups that take turns, 333 us; priority to the softmax, 336; priority by the wave's slot, 331.)
// FIXED: a row's softmax offset stays at the largest score of the first tile (no row maximum and no rescale decision in the loop:
// 8 % of one frame against 21, 9 % of three over 4 bits, 7 % of prompts under a window). Exact as long as nothing overflows or
// vanishes, which is checked before anything is stored: the sum of every row that sees a key of the walk within 2^-60 .. 2^100 and
// its values finite, or the workgroup makes the pass again with the running maximum and an eye on values that are not finite
// (returns false).
template <int D, bool FOUR, bool FIXED, class Params>
FV_DEV bool paged_tiles_item(const Params& p, const int wave, const int lane, const int block) {
    using G = TileGeo<D>;
    constexpr int kNO = D / 16, kTile = G::kTile;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    lds_u8* smem = (lds_u8*)smem_raw;
    const int q4 = lane >> 4, i16 = lane & 15;
    // The items lie in runs of 2^xcds XCDs, key head by key head, so that an L2 holds few heads' keys; the XCDs of a run take its items in
    // turn, so that each has as many of the long walks as the others. (One prompt of 16 heads on one key head: XCDs with an eighth
    // each took as long as the one with the last rows.)
    const bool full = block < p.big_full;
    const int at = full ? block : block - p.big_full, of = full ? p.big_full : p.big_rest;
    // (The second 32 of an XCD's items backwards: its 32 units take the first ones in turn, and the same would have the longest each time.)
    const int nth = (at >> 3) ^ (!full && at >> 8 == 1 ? 31 : 0);
    const int run = ((of << p.xcds) + 7) >> 3, in_run = (nth << p.xcds) + (at & ((1 << p.xcds) - 1));
    int item = ((at & 7) >> p.xcds) * run + in_run, chunk = 0;
    if (in_run >= run || item >= of) return true;
    if (!full) {
        // all tiles of a key head in their first share, then all in their second: neighbours walk the same keys, and the shares that
        // short walks do not have lie together (tile by tile they came to the same units again and again)
        const int set = paged_quot(item, p.big_set_shares), rest = item - set * p.big_set_shares.by;
        chunk = paged_quot(rest, p.big_set);
        item = p.big_full + set * p.big_set.by + rest - chunk * p.big_set.by;
    }
    const int cut_tile = item - p.big_full;   // (where it is cut)
    const int kvh = paged_quot(item, p.big_pieces.n);
    const PagedPiece piece = paged_piece<kBigRows>(p.big_pieces, p.b, p.group.by, (kvh + 1) * p.big_pieces.n.by - 1 - item);
    const int seq = piece.seq, tile = piece.tile;
    const PagedSeq sq = paged_seq(p.b, seq);
    const int rows = sq.count * p.group.by, row0 = tile * kBigRows;
    if (row0 >= rows || rows <= p.few) return true;
    const PagedWalk<kPart> w = paged_walk<kPart>(p, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kBigRows, rows) - 1, p.group));
    const int tiles = (w.n + 3) >> 2, e0 = chunk * p.big_chunk.by, e1 = full ? tiles : min(tiles, e0 + p.big_chunk.by);
    if (chunk > 0 && e0 >= e1) return true;
    const bool split = !full && tiles > p.big_chunk.by;
    const float sl2 = p.sl2;

    // the wave's rows: the keys that all of them see, those of one of them a lane (row lane % 32; exchanged where a tile asks)
    const int wrow = row0 + 32 * wave;
    PagedSight all_see = {0x7fffffff, 0, 0x7fffffff}, mine = {0, 0, 0};
    if (wrow < rows) {
        all_see = paged_all(p, sq, paged_quot(wrow, p.group), paged_quot(min(wrow + 32, rows) - 1, p.group));
        const int r = wrow + (lane & 31);
        mine = paged_sight(p, sq.first_pos() + paged_quot(min(r, rows - 1), p.group), sq.len);
    }
    // the parts of the walk that rows which all see `all` see whole: those before `a` and [b, c)
    struct Whole {
        int a, b, c;
        FV_DEV bool tile(int e) const { return 4 * e + 4 <= a || (4 * e >= b && 4 * e + 4 <= c); }
    };
    auto whole_parts = [&](const PagedSight& all) {
        auto before = [&](int t) { return min(t, w.ns) + min(max(t - w.b0, 0), w.n - w.ns); };   // of the parts before key 16 t
        return Whole{before(all.a / kPart), all.a >= all.lo ? 0 : before((all.lo + kPart - 1) / kPart), before(all.hi / kPart)};
    };
    const Whole whole = whole_parts(all_see);
    const int* table = p.b.table + (size_t)seq * p.b.table_stride;
    const int lg = p.pool.lg, slots = (1 << lg) - 1;
    // page numbers of 64 tiles of the walk, a tile a lane: that of the wave's 16 keys, and which of the tile's four 16 are in the pool
    int ids = 0, good = 0, ids_at = e0;
    bool clean = true;   // whether all of them are
    auto look_up = [&](int e) {
        ids_at = e;
        const int tile = min(e + lane, e1 - 1);
        good = 0;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int part = 4 * tile + x;
            const int id = table[w.key(min(part, w.n - 1)) >> lg];
            const bool ok = (unsigned)id < (unsigned)p.pool.pages;
            good |= ok || part >= w.n ? 1 << x : 0;   // (parts past the walk's end hold no key: none is seen)
            if (x == wave) ids = ok && part < w.n ? id : -1;
        }
        clean = __builtin_amdgcn_ballot_w64(good != 15) == 0;
    };
    // (the table, the queries and the first keys on their way together: short walks are mostly this wait)
    if (e0 < e1) look_up(e0);
    bf16x8 qf[D / 32][2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = wrow + 16 * g + i16, t = paged_quot(r, p.group);
        const uint16_t* q = p.q + (size_t)(sq.start + t) * p.q_stride + (kvh * p.group.by + r - t * p.group.by) * D + 8 * q4;
#pragma unroll
        for (int dk = 0; dk < D / 32; dk++) {
            u32x4 x = {0u, 0u, 0u, 0u};
            if (r < rows) x = *reinterpret_cast<const u32x4*>(q + 32 * dk);
            qf[dk][g] = __builtin_bit_cast(bf16x8, x);
        }
    }
    const TileReadBases rb = tile_read_bases<D>(lane);
    auto kbuf = [&](int m) -> lds_u8* { return smem + (m & 1) * kTile; };
    auto vbuf = [&](int m) -> lds_u8* { return smem + (2 + (m & 1)) * kTile; };
    // Where the wave's 16 keys of walk position e lie: their first key, its row in the pool, and how many of them, from the
    // front, are keys of the sequence in a page of the pool.
    struct Part {
        int key;
        unsigned row;
        int count;
    };
    auto part_of = [&](int e) {
        Part x;
        const int tile = min(e, e1 - 1), id = __builtin_amdgcn_readlane(ids, tile - ids_at);
        x.key = w.key(4 * tile + wave);   // (past the walk's end: no page, no key)
        x.row = (((unsigned)max(id, 0) * (unsigned)p.pool.kv_heads + (unsigned)kvh) << lg) + (unsigned)(x.key & slots);
        x.count = id < 0 ? 0 : min(max(w.any.hi - x.key, 0), 16);
        return x;
    };
    // Whether no row sees row r of a part: a key between the sink and the window. What lies there may be anything: scores that
    // are not seen are replaced, but values times a probability of 0 have to be numbers.
    auto some_hidden = [&](const Part& x) { return x.key < w.any.lo && x.key + 16 > w.any.a && w.any.a < w.any.lo; };
    auto hidden = [&](const Part& x, int r) { return x.key + r >= w.any.a && x.key + r < w.any.lo; };

    // bf16 pages
    constexpr int kIter = FOUR ? 2 : TileDma<4, D>::ITER, kUnits = kIter / 2;
    unsigned koff[kIter], voff[kIter];
    // 4-bit pages: the lane's quarter of row lane / 4
    constexpr int kQuarter = D / 32;   // words of codes; 16-byte pieces of bf16
    typedef __attribute__((ext_vector_type(kQuarter))) unsigned quarter;
    quarter kq = {}, vq = {};
    unsigned kqs = 127, vqs = 127;
    const int qrow = lane >> 2, qpart = lane & 3;
    if constexpr (!FOUR) {
#pragma unroll
        for (int it = 0; it < kIter; it++) {
            const int r = it * G::kRowsPerDma + lane / G::kChunks, c = lane % G::kChunks;
            koff[it] = r * G::kRow + ((c ^ G::kswz(r)) << 4) - (it & 1) * 1024;
            voff[it] = r * G::kRow + ((c ^ G::vswz(r)) << 4) - (it & 1) * 1024;
        }
    }
    // bf16: unit u (two loads) of the wave's part of a tile
    auto issue = [&](const void* pages, const Part& x, lds_u8* buf, const unsigned (&off)[kIter], int u) {
        const u32x4 desc = plane_descriptor((const uint8_t*)pages + (size_t)x.row * G::kRow, (unsigned)x.count * G::kRow);
        const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(size_t)(buf + wave * 16 * G::kRow + u * 2048));
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                     "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 lds"
                     :: "s"(m0), "v"(off[2 * u]), "v"(off[2 * u + 1]), "s"(desc) : "memory");
    };
    // 4 bits: the lane's quarter of K or V of a part, into registers ...
    auto fetch = [&](const void* pages, const uint8_t* scales, const Part& x, quarter& c, unsigned& sc) {
        const size_t row = (size_t)x.row + qrow;
        c = *reinterpret_cast<const quarter*>((const uint8_t*)pages + row * (D / 2) + qpart * (D / 8));
        sc = scales[row * (D / 32) + qpart * (D / 32) / 4];
    };
    auto clear = [&](lds_u8* buf, const Part& x) {   // bf16: hidden rows of the wave's part of a V tile
#pragma unroll
        for (int i = 0; i < 16 * G::kRow / 1024; i++) {
            const int r = i * G::kRowsPerDma + lane / G::kChunks;
            if (hidden(x, r)) lds_write_b128(buf + (16 * wave + r) * G::kRow + (lane % G::kChunks << 4), u32x4{0u, 0u, 0u, 0u});
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);
    };
    auto keep = [&](const Part& x, quarter& c, unsigned& sc) {   // 4 bits: values that nobody sees
        const bool none = qrow >= x.count || hidden(x, qrow);
#pragma unroll
        for (int j = 0; j < kQuarter; j++) c[j] = none ? 0u : c[j];
        sc = none ? 127u : sc;
    };
    // ... and piece j (8 channels) of it as bf16 to its place in the tile
    auto put = [&](lds_u8* buf, int swz, const quarter& c, unsigned sc, int j) {
        lds_write_b128(buf + (16 * wave + qrow) * G::kRow + (((kQuarter * qpart + j) ^ swz) << 4), fp4_eight(c[j], e8m0_scale(sc)));
    };

    f32x4 o[kNO][2], s_init[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    SoftmaxOffState st;
    st.init();
    ProbTile pb;

    // The second pass, a tile that some of the workgroup's rows see a part of: a value that is not finite belongs to the rows that see
    // it, whatever its weight, and a probability of zero does not keep it from the others. Such keys leave the V tile, and the rows
    // that see one add their share of it from the pool. (The first pass ends in the check where there is such a value.)
    const Whole wg_whole = whole_parts(paged_all(p, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kBigRows, rows) - 1, p.group)));
    auto set_apart = [&](int m, int e, const ProbTile& pb, f32x4 (&o)[kNO][2]) {
        lds_u8* mine_v = vbuf(m) + 16 * wave * G::kRow;
        unsigned bad_rows = 0;   // of the wave's 16
#pragma unroll
        for (int i = 0; i < 16 * G::kRow / 1024; i++) {
            lds_u8* at = mine_v + i * 1024 + lane * 16;
            const u32x4 v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(at);
            float bad = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) bad = not_finite(v[x], bad);
            const unsigned long long lanes = __builtin_amdgcn_ballot_w64(bad != 0.f);
#pragma unroll
            for (int r = 0; r < G::kRowsPerDma; r++)
                if ((lanes >> (r * G::kChunks)) & ((1ull << G::kChunks) - 1)) bad_rows |= 1u << (i * G::kRowsPerDma + r);
            if ((bad_rows >> (i * G::kRowsPerDma + lane / G::kChunks)) & 1) lds_write_b128(at, u32x4{0u, 0u, 0u, 0u});
        }
        auto* said = (__attribute__((address_space(3))) unsigned*)kbuf(m);   // (read by every wave, not yet loaded anew)
        if (lane == 0) said[wave] = bad_rows;
        __builtin_amdgcn_s_waitcnt(0xC07F);
        block_barrier();
        const u32x4 of = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(said);
        unsigned long long keys = 0;
#pragma unroll
        for (int x = 0; x < 4; x++) keys |= (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane(of[x]) << (16 * x);
#pragma unroll 1
        for (; keys != 0; keys &= keys - 1) {
            const int x = __builtin_ctzll(keys), key = w.key(min(4 * e + (x >> 4), w.n - 1)) + (x & 15);
            const int id = table[key >> lg];
            const unsigned row = (((unsigned)max(id, 0) * (unsigned)p.pool.kv_heads + (unsigned)kvh) << lg) + (unsigned)(key & slots);
            float pj[2];
#pragma unroll
            for (int g = 0; g < 2; g++) {   // key x: the (x & 3)-th of its four of block (x >> 4) & 1 in lanes 16 ((x >> 2) & 3) ..
                const u32x4 lo = __builtin_bit_cast(u32x4, pb[0][g]), hi = __builtin_bit_cast(u32x4, pb[1][g]);
                const u32x4 half = x < 32 ? lo : hi;
                const unsigned pair = (x & 16) ? ((x & 2) ? half[3] : half[2]) : ((x & 2) ? half[1] : half[0]);
                pj[g] = __shfl(__builtin_bit_cast(float, x & 1 ? pair & 0xffff0000u : pair << 16), 16 * ((x >> 2) & 3) + i16, 64);
                const PagedSight row_sees = {__shfl(mine.a, 16 * g + i16, 64), __shfl(mine.lo, 16 * g + i16, 64), __shfl(mine.hi, 16 * g + i16, 64)};
                if (pj[g] == 0.f && row_sees.one(key)) pj[g] = kLeast;
            }
#pragma unroll
            for (int db = 0; db < kNO; db++) {
                float v[4];
                pool_values<D, FOUR>(p.pool, row, 16 * db + 4 * q4, v);
#pragma unroll
                for (int g = 0; g < 2; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[db][g][i] += pj[g] == 0.f ? 0.f : pj[g] * v[i];
            }
        }
        __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0), lgkmcnt(0)
        block_barrier();
    };
    auto mask_tile = [&](ScoreTile& s, int e) {
        if (whole.tile(e) && clean) return;
        const int ok = __builtin_amdgcn_readlane(good, e - ids_at);
        const unsigned m[3] = {(unsigned)mine.a, (unsigned)mine.lo, (unsigned)mine.hi};
        int both[3][2];   // the even rows of 16 lanes hold block 0's, the odd ones block 1's
#pragma unroll
        for (int x = 0; x < 3; x++) {
            const auto r = __builtin_amdgcn_permlane16_swap(m[x], m[x], false, false);
            both[x][0] = (int)r[0];
            both[x][1] = (int)r[1];
        }
        auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };   // bits of the first n of 4 keys
#pragma unroll
        for (int kb = 0; kb < 4; kb++) {
            const bool none = 4 * e + kb >= w.n || !((ok >> kb) & 1);
            const int at = (none ? 0x7fffff00 : w.key(4 * e + kb)) + 4 * q4;   // (past every key: a table holds fewer than 2^31)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const unsigned bits = below(both[0][g] - at) | (below(both[2][g] - at) & ~below(both[1][g] - at));
#pragma unroll
                for (int i = 0; i < 4; i++) s[kb][g][i] = (bits >> i) & 1 ? s[kb][g][i] : neg_inf();
            }
        }
    };

    if (e0 < e1) {
        Part cur = part_of(e0), next = part_of(e0 + 1);   // of the tile whose V is loaded next, whose K is
        if constexpr (FOUR) {
            fetch(p.pool.k, p.pool.ks, cur, kq, kqs);
#pragma unroll
            for (int j = 0; j < kQuarter; j++) put(kbuf(0), G::kswz(qrow), kq, kqs, j);
            fetch(p.pool.v, p.pool.vs, cur, vq, vqs);
            fetch(p.pool.k, p.pool.ks, next, kq, kqs);
            __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
            __builtin_amdgcn_sched_barrier(0);
        } else {
#pragma unroll
            for (int u = 0; u < kUnits; u++) issue(p.pool.k, cur, kbuf(0), koff, u);
        }
#pragma unroll
        for (int dk = 0; dk < D / 32; dk++) asm volatile("" : "+v"(qf[dk][0]), "+v"(qf[dk][1]));   // (waited for here, not among the tile loads)
        if constexpr (!FOUR) wait_vmcnt<0>();
        block_barrier();
        constexpr int kAhead = 3;
        auto phase = [&](int m, auto first) {
            const int e = e0 + m;
            Part after = next;
            ScoreTile s;
            auto hook = [&](int i) {
                if constexpr (FOUR) {
                    // V of this tile and K of the next, fetched a phase ago; then the fetches for the next phase
                    if (i == 0) keep(cur, vq, vqs);
                    if (i < kQuarter) put(vbuf(m), G::vswz(qrow), vq, vqs, i);
                    else if (i < 2 * kQuarter) put(kbuf(m + 1), G::kswz(qrow), kq, kqs, i - kQuarter);
                    else if (i == 2 * kQuarter) after = part_of(e + 2), fetch(p.pool.v, p.pool.vs, next, vq, vqs);
                    else if (i == 2 * kQuarter + 1) fetch(p.pool.k, p.pool.ks, after, kq, kqs);
                } else {
                    if (i < kUnits) issue(p.pool.v, cur, vbuf(m), voff, i);
                    else if (i < 2 * kUnits) issue(p.pool.k, next, kbuf(m + 1), koff, i - kUnits);
                    else if (i == 2 * kUnits) after = part_of(e + 2);
                }
            };
            __builtin_amdgcn_s_setprio(1);
            if constexpr (first()) {
                mfma_phase<false, kAhead, D>(vbuf(0), kbuf(0), rb, pb, o, qf, s, s_init, hook);
                if constexpr (FOUR) {   // (a phase without its P V part has half the gaps)
#pragma unroll
                    for (int i = G::kKGroups; i < 2 * kQuarter + 2; i++) hook(i);
                }
#pragma unroll
                for (int db = 0; db < kNO; db++) o[db][0] = o[db][1] = f32x4{0.f, 0.f, 0.f, 0.f};
            } else {
                mfma_phase<true, kAhead, D>(vbuf(m - 1), kbuf(m), rb, pb, o, qf, s, s_init, hook);
            }
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            mask_tile(s, e);
            if constexpr (first()) softmax_first_off<true>(s, st, s_init, sl2, pb);
            else if constexpr (FIXED) softmax_off_tile<true>(s, st, sl2, pb);
            else softmax_tile_off<true>(s, st, o, s_init, sl2, pb);
            asm volatile("" ::"v"(pb[0][0]), "v"(pb[0][1]), "v"(pb[1][0]), "v"(pb[1][1]), "v"(st.l_acc[0]), "v"(st.l_acc[1]));
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (FOUR) {
                __builtin_amdgcn_s_waitcnt(0xC07F);
            } else {
                wait_vmcnt<0>();
                if (some_hidden(cur)) clear(vbuf(m), cur);
            }
            cur = next;
            next = after;
            block_barrier();   // K(m + 1), V(m) resident; this phase's tiles read by every wave
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!FIXED) {
                if (!wg_whole.tile(e)) set_apart(m, e, pb, o);
            }
        };
        phase(0, std::true_type{});
#pragma unroll 1
        for (int m = 1; m < e1 - e0; m++) {
            if (e0 + m + 2 - ids_at >= 64 && e0 + m + 2 < e1) look_up(e0 + m);
            phase(m, std::false_type{});
        }
        pv_tile<D>(vbuf(e1 - e0 - 1), rb.v, pb, o);
    } else {
#pragma unroll
        for (int db = 0; db < kNO; db++) o[db][0] = o[db][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    if constexpr (FIXED) {
        // the lane's part of its rows' check; a row without a key in the walk has a sum of zero by right
        const int p0 = 4 * e0, p1 = min(4 * e1, w.n);   // the parts; those past the sink hold keys [from, to)
        const int from = w.key(max(p0, w.ns)), to = w.key(max(p1 - 1, 0)) + kPart;
        const bool any = p0 < p1 && wrow + (lane & 31) < rows &&
                         ((p0 < w.ns && p0 * kPart < mine.a) || (p1 > w.ns && (max(mine.lo, from) < min(mine.hi, to) || from < mine.a)));
        const auto sees = __builtin_amdgcn_permlane16_swap((unsigned)any, (unsigned)any, false, false);   // (exchanged as in mask_tile)
        float chk = 0.f;
        bool fine = true;
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const float l = quad_sum(st.l_acc[g]);
            fine = fine && (wrow + 16 * g + i16 >= rows || (l < 0x1p+100f && (l > 0x1p-60f || (l == 0.f && !sees[g]))));
#pragma unroll
            for (int db = 0; db < kNO; db++)
#pragma unroll
                for (int i = 0; i < 4; i++) chk = __builtin_fmaf(o[db][g][i], 0.f, chk);
        }
        // (of rows past the last nothing is stored; their values are those of queries of zeros)
        const bool wave_ok = wrow >= rows || __builtin_amdgcn_ballot_w64(!(fine && chk == 0.f)) == 0;
        auto* votes = (__attribute__((address_space(3))) unsigned*)(smem + kTile);   // (K buffer 1: the last P V reads none, and a second pass writes it behind its first barrier)
        if (lane == 0) votes[wave] = wave_ok ? 0u : 1u;
        __builtin_amdgcn_s_waitcnt(0xC07F);
        block_barrier();
        const u32x4 v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(votes);
        if (__builtin_amdgcn_readfirstlane(v[0] | v[1] | v[2] | v[3]) != 0) return false;
    }
    const size_t shares = (size_t)chunk * p.big_rows + (size_t)cut_tile * kBigRows;
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const float l = quad_sum(st.l_acc[g]);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int r = wrow + 16 * g + i16, t = paged_quot(r, p.group);
        if (r >= rows) continue;
        const size_t dst = (size_t)(sq.start + t) * p.heads + kvh * p.group.by + (r - t * p.group.by);
        const size_t share = shares + (r - row0);
        if (split && q4 == 0) p.big_lse[share] = l == 0.f ? neg_inf() : st.log2_offset<true>(g, sl2) + __log2f(l);
#pragma unroll
        for (int db = 0; db < kNO; db++) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = o[db][g][i] * inv;
            const size_t at = dst * D + 16 * db + 4 * q4;
            if (split) *reinterpret_cast<f32x4*>(p.big_o + share * D + 16 * db + 4 * q4) = x;
            else if (p.out_is_bf16) *reinterpret_cast<bf16x4*>((uint16_t*)p.out + at) = __builtin_convertvector(x, bf16x4);
            else *reinterpret_cast<f32x4*>((float*)p.out + at) = x;
        }
    }
    return true;
}
// The kernel's arguments read again from their segment, of which PagedAttnParams is the whole, and the lane counted anew, so that the
// second pass keeps nothing of the first in registers. It spills (65 - 184 registers where both share the kernel's 256, or 168 at 64
// channels) and the first does not in its loop. Where every workgroup needs it, a call takes 3 times as long over bf16 pages, 5 over
// 4 bits (keys whose scores grow by 1000 and more along a sequence): a frame of 1560 rows x 12 heads on 32760 298 -> 929 us, prompts under a window
// 229 -> 702, three frames of two sequences over 4 bits 1.75 -> 9.0 ms.
template <int D, bool FOUR>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void paged_tiles_kernel(const PagedAttnParams p) {
    int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = blockIdx.x;
    if (paged_tiles_item<D, FOUR, true>(p, wave, threadIdx.x & 63, block)) return;
    using ConstParams = const __attribute__((address_space(4))) PagedAttnParams;
    ConstParams* again = (ConstParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(again));
    int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane), "+s"(wave), "+s"(block));
    paged_tiles_item<D, FOUR, false>(*again, wave, lane, block);
}

// The shares of a split walk joined: out = sum_c w_c O_c / sum_c w_c, w_c = 2^(lse_c - max lse). G groups of D / 4 threads share a
// row's shares out, four at a time each, with a running maximum, and meet in LDS; rows whose walk one workgroup made have
// their result already. A row with many shares is a chain of waits, so G = 8 then (61 shares of one token's 40 heads: 4.0
// us); few shares are the memory's to bound, and G = 1 keeps them out of LDS (three of 1560 rows x 12 heads: 8.5 us).
template <int D, int G>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnParams p) {
    constexpr int kPer = D / 4, kRows = 256 / (kPer * G);
    __shared__ float lds_top[kRows][G], lds_sum[kRows][G];
    __shared__ f32x4 lds_acc[kRows][G][kPer];
    constexpr int kPerTile = kBigRows / kRows;
    const int slot = threadIdx.x / (kPer * G), gi = threadIdx.x / kPer % G, c = threadIdx.x % kPer;
    const bool few = (int)blockIdx.x >= p.join_tiles;
    int kvh, seq, r, item = 0;
    if (few) {
        const int at = blockIdx.x - p.join_tiles, q = paged_quot(at, p.join_few);
        seq = paged_quot(q, p.kv_heads);
        kvh = q - seq * p.kv_heads.by;
        r = (at - q * p.join_few.by) * kRows + slot;
    } else {
        item = p.big_full + blockIdx.x / kPerTile;   // (as paged_tiles_item counts)
        kvh = paged_quot(item, p.big_pieces.n);
        const PagedPiece piece = paged_piece<kBigRows>(p.big_pieces, p.b, p.group.by, (kvh + 1) * p.big_pieces.n.by - 1 - item);
        seq = piece.seq;
        r = piece.tile * kBigRows + (blockIdx.x % kPerTile) * kRows + slot;
    }
    const PagedSeq sq = paged_seq(p.b, seq);
    const int rows = sq.count * p.group.by, t = paged_quot(r, p.group);
    const size_t dst = (size_t)(sq.start + t) * p.heads + kvh * p.group.by + (r - t * p.group.by);
    int chunks = 0;
    size_t first = 0, step = 0;   // the row's place in the first share, rows to the next
    if (r < rows && few == (rows <= p.few)) {
        auto shares = [&](const auto& walk, int parts, const PagedDiv& chunk) { return paged_quot((walk.n + parts - 1) / parts + chunk.by - 1, chunk); };
        if (few) {
            const int row0 = r & -p.rows_m;
            first = ((size_t)seq * p.kv_heads.by + kvh) * p.few + r;
            step = (size_t)p.b.seqs * p.kv_heads.by * p.few;
            chunks = shares(paged_walk<kStep>(p, sq, paged_quot(row0, p.group), paged_quot(min(row0 + p.rows_m, rows) - 1, p.group)), 1, p.rows_chunk);
        } else {
            const int row0 = r & -kBigRows;
            chunks = shares(paged_walk<kPart>(p, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kBigRows, rows) - 1, p.group)), 4, p.big_chunk);
            first = (size_t)(item - p.big_full) * kBigRows + (r - row0);
            step = (size_t)p.big_rows;
        }
    }
    if (G == 1 && chunks <= 1) return;
    const float* part_o = few ? p.rows_o : p.big_o;
    const float* part_lse = few ? p.rows_lse : p.big_lse;
    float top = neg_inf(), total = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (chunks > 1) {
        for (int s = gi; s < chunks; s += 4 * G) {
            float lse[4];
            f32x4 x[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const size_t at = (size_t)min(s + u * G, chunks - 1) * step + first;
                lse[u] = part_lse[at];
                x[u] = *reinterpret_cast<const f32x4*>(part_o + at * D + 4 * c);
            }
            float m = top;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (s + u * G >= chunks) lse[u] = neg_inf();
                m = __builtin_fmaxf(m, lse[u]);
            }
            const float k = top == neg_inf() ? 0.f : fast_exp2(top - m);
            total *= k;
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] *= k;
#pragma unroll
            for (int u = 0; u < 4; u++) {   // (a share without a key has -inf; one whose sum is not a number makes the row that)
                const float k = lse[u] == neg_inf() ? 0.f : fast_exp2(lse[u] - m);
                total += k;
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i] += lse[u] == neg_inf() ? 0.f : k * x[u][i];
            }
            top = m;
        }
    }
    if constexpr (G > 1) {
        if (c == 0) lds_top[slot][gi] = top, lds_sum[slot][gi] = total;
        lds_acc[slot][gi][c] = acc;
        __syncthreads();
        if (chunks <= 1 || gi != 0) return;
        float m = neg_inf();
#pragma unroll
        for (int x = 0; x < G; x++) m = __builtin_fmaxf(m, lds_top[slot][x]);
        total = 0.f, acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < G; x++) {
            const float k = lds_top[slot][x] == neg_inf() ? 1.f : fast_exp2(lds_top[slot][x] - m);   // (-inf: zeros, or not a number)
            total += k * lds_sum[slot][x];
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] += k * lds_acc[slot][x][c][i];
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] *= inv;
    if (p.out_is_bf16) *reinterpret_cast<bf16x4*>((uint16_t*)p.out + dst * D + 4 * c) = __builtin_convertvector(acc, bf16x4);
    else *reinterpret_cast<f32x4*>((float*)p.out + dst * D + 4 * c) = acc;
}

// Steps of `step` keys that the walk of a tile of `rows` rows may have. (Host arithmetic on the call's bounds: the lengths
// themselves are the device's.)
size_t walk_bound(size_t step, size_t rows, size_t group, size_t max_len, size_t block_tokens, size_t window, size_t sink) {
    size_t steps = (max_len + step - 1) / step;
    if (window > 0) {   // the first token's window and the blocks to the last token's, a step more (they begin anywhere in one); the sink
        const size_t apart = (rows + group - 2) / group, blocks = window + (apart + block_tokens - 1) / block_tokens, far = (size_t)1 << 31;
        const size_t band = blocks < far / block_tokens ? blocks * block_tokens : far, keep = sink < far / block_tokens ? sink * block_tokens : far;
        steps = std::min(steps, (band + step - 1) / step + 1 + (keep + step - 1) / step);
    }
    return std::max<size_t>(steps, 1);
}

constexpr size_t kMostShares = (size_t)1 << 30;   // bytes of a kernel's shares: past it its walks are cut less
// How a call is cut.
struct PagedCut {
    size_t few = 0;                         // rows a key head up to which a sequence is paged_rows_kernel's
    size_t nt = 0;                          // its tiles of 16 rows; 0: not launched
    size_t rows_tiles = 1, rows_chunk = 1, rows_chunks = 1;
    PagedPieces big = {};                   // of paged_tiles_kernel, a key head; none: not launched
    size_t big_full = 0, big_chunk = 1, big_chunks = 1;
    size_t chunks() const { return std::max(nt ? rows_chunks : 1, big.n.by ? big_chunks : 1); }
};
// bf16: two tiles of 16 rows cost paged_rows_kernel a second pass over the keys' operands, or a second walk, and paged_tiles_kernel, which
// pads to 128, streams the keys as fast (48 sessions of 5 drafts x 4 heads, a window of 2048: 86 us by rows, 77.5 by tiles; 16 x 8 x 5
// heads, 8000 tokens: 160, 108; single tokens of 5 heads: 240, 242). 4 bits: the tiles' arithmetic is the bound (single tokens 177 us by
// rows, 492 by tiles; 40 rows the same, 73).
constexpr size_t few_rows(bool four) { return four ? 64 : 16; }
PagedCut paged_cut(size_t heads, size_t kv_heads, size_t d, bool four, size_t seqs, size_t tokens, size_t max_q, size_t max_len, size_t block_tokens,
                   size_t window, size_t sink) {
    PagedCut c;
    const size_t group = heads / kv_heads, rows = max_q * group, units = (size_t)fv_compute_units(), most_few = few_rows(four);
    if (rows > most_few) {
        const size_t tiles = (rows + kBigRows - 1) / kBigRows;   // (of the longest)
        c.big = paged_pieces(kBigRows, seqs, tokens, max_q, group);
        const size_t steps = (walk_bound(kPart, kBigRows, group, max_len, block_tokens, window, sink) + 3) / 4;
        // Shares of the walk, by microseconds (fitted to 446 calls in 1 to 24 shares, within 7 %; the number that it takes is 1 % slower than
        // the best of them on average): rounds of as many workgroups as there is room for, each step by how many a unit has at once, or
        // by what the memory takes where few tiles share their keys; against a launch and the bytes that joining moves. Where the last
        // round is far from full, the tiles of the rounds before keep their walk whole and only the rest are cut. Tiles whose walks
        // differ (causal, or of ragged prompts) fill the rounds by themselves: their steps in all, and the longest at the end. One frame
        // of 1560 against 32760, 12 heads: in 1, 2, 3, 4 shares 538, 427, 290, 362 us.
        const size_t numbers = kv_heads * (size_t)c.big.n.by;
        const size_t slots = (d == 64 ? 3 : 2) * (units / 8 * 8);
        const bool ragged = c.big.tiles.by == 0;
        const size_t held = ragged ? kv_heads * (tokens * group / kBigRows + 1) : numbers;   // (the numbers without those that may be unused)
        const bool in_window = steps < (max_len / kPart + 3) / 4;
        const double later = block_tokens < max_q && max_q <= max_len ? (double)(max_q - block_tokens) : 0.0;   // rows behind the first block's
        const double mean = in_window ? 1.0 : ragged ? 0.6 : 1.0 - 0.5 * later / (double)max_len;   // of the longest walk
        const bool varied = ragged || mean < 0.8;
        auto steps_us = [&](double n, double wgs) {
            const int at_once = wgs <= (double)units ? 0 : wgs <= 2.0 * (double)units ? 1 : 2;
            const double wide[] = {1.07, 1.49, 1.49}, narrow[] = {0.67, 0.97, 1.26}, bytes = 64.0 * (double)(four ? d + d / 16 : 4 * d);
            return n * std::max((d == 64 ? narrow : wide)[at_once] * (four ? 1.08 : 1.0), wgs / (double)tiles * bytes / (at_once == 0 ? 5e6 : 6.1e6));
        };
        double best = 0;
        const size_t rounds_before = varied ? 0 : held / slots;
        for (size_t keep = 0; keep <= std::min<size_t>(rounds_before, 2); keep++) {
            const size_t full = keep == 0 ? 0 : (rounds_before - (keep - 1)) * slots, rest = held - full;   // (full only where walks are alike: held is numbers)
            if (rest == 0) continue;
            for (size_t k = 1; k <= 64 && k <= steps; k++) {
                const size_t chunk = (steps + k - 1) / k, shares = (steps + chunk - 1) / chunk, wgs = rest * shares;
                if (k > 1 && shares > kMostShares / ((numbers - full) * kBigRows * d * 4)) break;
                double cost = (double)(full / slots) * steps_us((double)steps, (double)slots);
                if (varied) {
                    const double each = std::max(1.0, (double)shares * mean), all = (double)rest * each, at_once = std::min(all, (double)slots);
                    cost += std::max(all / (double)slots * steps_us((double)steps * mean / each, at_once) + steps_us(0.43 * (double)chunk, at_once) * at_once / (double)slots,
                                     steps_us(0.92 * (double)chunk, at_once));
                } else {
                    cost += (double)(wgs / slots) * steps_us((double)chunk * mean, (double)slots) + steps_us((double)chunk * mean, (double)(wgs % slots)) * (wgs % slots != 0);
                }
                if (shares > 1)
                    cost += 2.0 + (double)(shares * std::min(rest * kBigRows, tokens * heads)) * std::min(1.0, mean + 0.1) * 8.0 * (double)d / 5.5e6 + 0.01 * (double)(numbers - full);
                if ((keep == 0 && k == 1) || cost < 0.97 * best) best = cost, c.big_full = full, c.big_chunk = chunk, c.big_chunks = shares;
            }
        }
        if (c.big_chunks == 1) c.big_full = 0;
    }
    // (Sequences of few rows beside longer ones: a launch of their own where they may be many, by the mean, and then for those of one
    // tile of rows; else they are the tiles', which take any, and the launch, 5 us, is saved.)
    if (rows <= most_few || 2 * tokens < seqs * max_q) {
        const size_t most = rows <= most_few ? rows : 16;
        c.few = most;
        c.nt = most <= 16 ? 1 : 2;
        c.rows_tiles = (most + 16 * c.nt - 1) / (16 * c.nt);
        const size_t steps = walk_bound(kStep, 16 * c.nt, group, max_len, block_tokens, window, sink);
        // Shares of up to 128 steps, so that long sequences among short ones are cut (40 sessions of 15 to 100 % of 32760 tokens, 8
        // key heads, 4 bits: whole 270 us, 256 steps 211, 128 180, 64 184), a walk of up to 192 whole (128 sessions under a
        // window of 4096: 100 us, in two 115). Where that leaves units idle, as many shares as give each unit one workgroup, two over 4
        // bits: 8 sessions of 12 heads x 6000 tokens in bf16, 96 workgroups 71 us, 192 49; 2 of 20000 x 12, 240 workgroups 42, 264 50 (some
        // units have two). A share costs its launch and its join some 4 us where a step of each wave costs 1, so short walks are cut in three
        // or more (one of 1500 tokens, 40 / 8 heads: whole 17.7, 11 shares 10.4; 30 of 1400 over 4 bits whole 15.2, in two 17.0) or not at all.
        const size_t base = seqs * kv_heads * c.rows_tiles;
        size_t shares = steps <= 192 ? 1 : (steps + 127) / 128;
        const size_t fill = std::min((four ? 2 : 1) * units / base, std::max(steps / 8, std::min<size_t>(steps / 4, 16)));
        if (steps >= 36 && fill >= (steps < 96 ? 3 : 2)) shares = std::max(shares, fill);
        // (max_len is a bound that lengths may be far below. 256 sequences of 9 drafts, 32 / 8 heads, over 4 bits, 500 to 30000 keys: under
        // a bound of 2^20 9.7 GB of shares of 128 steps 2.89 ms, a gigabyte 3.31, its walks being whole; of 12 drafts, 40 / 8 heads, under 2^17
        // 2.03 GB 2.20 ms, a gigabyte 1.98.)
        shares = std::min(shares, std::max<size_t>(kMostShares / (seqs * kv_heads * c.few * d * 4), 1));
        size_t chunk = ((steps + shares - 1) / shares + kWaves - 1) / kWaves * kWaves;
        c.rows_chunk = chunk;
        c.rows_chunks = (steps + chunk - 1) / chunk;
    }
    return c;
}
// The shares' places in the workspace.
struct PagedParts {
    size_t rows_o = 0, rows_lse = 0, big_o = 0, big_lse = 0, big_rows = 0, bytes = 0;   // rows_o ..: bytes from its start
    PagedParts(const PagedCut& c, size_t seqs, size_t kv_heads, size_t d) {
        auto take = [this](size_t n) {
            const size_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        if (c.nt && c.rows_chunks > 1) {
            const size_t rows = seqs * kv_heads * c.few;
            rows_o = take(c.rows_chunks * rows * d * 4), rows_lse = take(c.rows_chunks * rows * 4);
        }
        if (c.big.n.by && c.big_chunks > 1) {
            big_rows = (kv_heads * (size_t)c.big.n.by - c.big_full) * kBigRows;
            big_o = take(c.big_chunks * big_rows * d * 4), big_lse = take(c.big_chunks * big_rows * 4);
        }
    }
};

}  // namespace
}  // namespace fv

static bool mask_fits(size_t block_tokens, size_t window, size_t sink) {
    return std::max({block_tokens, window, sink}) <= (size_t)INT_MAX / 2;
}

extern "C" {

size_t fv_paged_attention_workspace_bytes_for(int four_bits, size_t heads, size_t kv_heads, size_t d, size_t seqs, size_t tokens, size_t max_q,
                                              size_t max_len, size_t block_tokens, size_t window, size_t sink) {
    if (kv_heads == 0 || heads < kv_heads || heads % kv_heads != 0 || block_tokens == 0 || seqs == 0 || tokens == 0 || max_q == 0) return 0;
    // (what fv_paged_attention refuses: products of these numbers would pass 64 bits)
    if ((d != 64 && d != 128) || heads > 65535 || seqs > kMostSeqs || tokens > kMostRows || max_len > (size_t)INT_MAX || !mask_fits(block_tokens, window, sink))
        return 0;
    const fv::PagedCut c = fv::paged_cut(heads, kv_heads, d, four_bits != 0, seqs, tokens, std::min(max_q, tokens), max_len, block_tokens, window, sink);
    return fv::PagedParts(c, seqs, kv_heads, d).bytes;
}
size_t fv_paged_attention_workspace_bytes(size_t heads, size_t kv_heads, size_t d, size_t seqs, size_t tokens, size_t max_q, size_t max_len,
                                          size_t block_tokens, size_t window, size_t sink) {
    size_t most = 0;
    for (const int four : {0, 1})
        most = std::max(most, fv_paged_attention_workspace_bytes_for(four, heads, kv_heads, d, seqs, tokens, max_q, max_len, block_tokens, window, sink));
    return most;
}

int fv_paged_attention(const uint16_t* q, size_t q_stride, void* out, int out_is_bf16, size_t heads, const void* k_pages,
                       const void* v_pages, const void* k_scales, const void* v_scales, size_t pages, size_t page_tokens, size_t kv_heads,
                       size_t d, const int32_t* q_start, const int32_t* lens, const int32_t* table, size_t table_stride, size_t table_pages,
                       size_t seqs, size_t tokens, size_t max_q, size_t max_len, float scale, size_t block_tokens, size_t window,
                       size_t sink, void* workspace, size_t workspace_bytes, void* stream) {
    if (seqs == 0 || tokens == 0 || max_q == 0) return FV_OK;   // (empty arrays may have no address)
    fv::PagedAttnParams p;
    const int rc = fv_paged_args("paged attention", k_pages, v_pages, k_scales, v_scales, pages, page_tokens, kv_heads, d, q_start, lens,
                                 table, table_stride, table_pages, seqs, tokens, &max_len, &p.pool, &p.b);
    if (rc != FV_OK) return rc;
    if (!q || !out) return fv_invalid("paged attention: null operand");
    if (heads == 0 || heads % kv_heads != 0) return fv_invalid("paged attention: query heads must be a multiple of the key heads");
    if (heads > 65535) return fv_decline("paged attention: too many heads");
    if (q_stride < heads * d) return fv_invalid("paged attention: tokens overlap (a stride below heads * d)");
    if (q_stride % 8 != 0 || q_stride > (size_t)INT_MAX / 4) return fv_decline("paged attention: the stride must be a multiple of 8 elements");
    if (((uintptr_t)q & 15) != 0 || ((uintptr_t)out & 15) != 0) return fv_invalid("paged attention: operands must be 16-byte aligned");
    if (!(scale > 0.f) || !(scale <= 2e38f)) return fv_decline("paged attention: scale must be positive and finite");
    if (block_tokens == 0) return fv_invalid("paged attention: block_tokens must be positive");
    if (!mask_fits(block_tokens, window, sink)) return fv_decline("paged attention: mask too large");
    if (max_q > tokens) max_q = tokens;
    const bool four = k_scales != nullptr;
    fv::PagedCut c = fv::paged_cut(heads, kv_heads, d, four, seqs, tokens, max_q, max_len, block_tokens, window, sink);
    fv::PagedParts parts(c, seqs, kv_heads, d);
    if (parts.bytes > 0 && (!workspace || workspace_bytes < parts.bytes)) {   // a share is the whole walk
        c.rows_chunk *= c.rows_chunks, c.big_chunk *= c.big_chunks;
        c.rows_chunks = c.big_chunks = 1, c.big_full = 0;
        parts = fv::PagedParts(c, seqs, kv_heads, d);
        workspace = nullptr;
    }
    const bool split = c.chunks() > 1;
    if (split && ((uintptr_t)workspace & 255) != 0) return fv_invalid("paged attention: the workspace must be 256-byte aligned");
    // eight groups of threads a row of the join, or one: where rows are few for their shares
    const size_t most_shares = c.big_chunks > 1 ? c.big_chunks : c.rows_chunks;
    const bool many = most_shares > 4 && tokens * heads < 128 * most_shares;
    const size_t group = heads / kv_heads;
    const int xcds = kv_heads % 8 == 0 ? 0 : kv_heads % 4 == 0 ? 1 : kv_heads % 2 == 0 ? 2 : 3;   // (a run has whole key heads)
    const size_t join_rows = 256 / (d / 4 * (many ? 8 : 1));   // a workgroup
    const size_t cut_tiles = c.big.n.by && c.big_chunks > 1 ? kv_heads * (size_t)c.big.n.by - c.big_full : 0;
    const size_t join_tiles = cut_tiles * (fv::kBigRows / join_rows), join_few = c.rows_chunks > 1 ? (c.few + join_rows - 1) / join_rows : 0;
    const size_t row_blocks = seqs * kv_heads * c.rows_tiles * c.rows_chunks, big_rest = (kv_heads * (size_t)c.big.n.by - c.big_full) * c.big_chunks;
    size_t an_xcd = (((big_rest << xcds) + 7) / 8 + ((size_t)1 << xcds) - 1) >> xcds;
    if (an_xcd > 32) an_xcd = std::max<size_t>(an_xcd, 64);   // (the second 32 are taken backwards)
    const size_t big_blocks = c.big_full + 8 * an_xcd, join_blocks = join_tiles + seqs * kv_heads * join_few;
    constexpr size_t kMost = (size_t)1 << 24;   // (a launch holds fewer than 2^32 work-items)
    if (row_blocks >= kMost || big_blocks >= kMost || (split && join_blocks >= kMost)) return fv_decline("paged attention: too large for one launch");
    p.q = q, p.q_stride = (long)q_stride, p.out = out, p.out_is_bf16 = out_is_bf16 != 0;
    p.heads = (int)heads, p.group = fv::paged_div(group), p.kv_heads = fv::paged_div(kv_heads);
    p.sl2 = (float)((double)scale * 1.4426950408889634);
    p.block_tokens = fv::paged_div(block_tokens), p.window = (int)window, p.sink = (int)sink;
    p.few = (int)c.few, p.rows_m = (int)(16 * c.nt);
    p.rows_tiles = fv::paged_div(c.rows_tiles), p.rows_chunk = fv::paged_div(c.rows_chunk), p.rows_chunks = fv::paged_div(c.rows_chunks);
    const size_t set = c.big_full ? kv_heads * (size_t)c.big.n.by - c.big_full : (size_t)c.big.n.by;   // (a key head's; else all)
    p.big_set = fv::paged_div(set), p.big_set_shares = fv::paged_div(set * c.big_chunks);
    p.big_chunk = fv::paged_div(c.big_chunk), p.big_pieces = c.big;
    p.join_tiles = (int)join_tiles, p.join_few = fv::paged_div(join_few);
    p.big_full = (int)c.big_full, p.big_rest = (int)big_rest, p.xcds = xcds;
    uint8_t* ws = (uint8_t*)workspace;
    p.rows_o = (float*)(ws + parts.rows_o), p.rows_lse = (float*)(ws + parts.rows_lse);
    p.big_o = (float*)(ws + parts.big_o), p.big_lse = (float*)(ws + parts.big_lse), p.big_rows = (long)parts.big_rows;
    hipStream_t st = (hipStream_t)stream;
    fv::paged_pick(d == 128, [&](auto d128) {
        fv::paged_pick(four, [&](auto f) {
            constexpr int D = d128() ? 128 : 64;
            if (c.big.n.by)
                hipLaunchKernelGGL((fv::paged_tiles_kernel<D, f()>), dim3((unsigned)big_blocks), dim3(256), 4 * fv::TileGeo<D>::kTile, st, p);
            if (c.nt == 1) hipLaunchKernelGGL((fv::paged_rows_kernel<D, f(), 1>), dim3((unsigned)row_blocks), dim3(256), 0, st, p);
            if constexpr (f())   // (the only pages whose calls have two tiles of rows, few_rows)
                if (c.nt == 2) hipLaunchKernelGGL((fv::paged_rows_kernel<D, true, 2>), dim3((unsigned)row_blocks), dim3(256), 0, st, p);
            if (split)
                fv::paged_pick(many, [&](auto m) { hipLaunchKernelGGL((fv::paged_join_kernel<D, m() ? 8 : 1>), dim3((unsigned)join_blocks), dim3(256), 0, st, p); });
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "paged_attention");
}

}  // extern "C"
