// Attention over packed sequences (declarations: include/fv_sdpa_hip.h): for every row (token t of a sequence, query head h),
// o = sum_j softmax_j(scale q . k_j) v_j over the keys j of its sequence that it sees, and lse = ln sum_j e^(scale q . k_j), which the
// gradients start from (packed_back.hip).
//
// Rows of one key head lie together (token by token, the heads of its group in turn), so a tile of keys serves a whole group, and a few
// tokens of many heads fill a tile of rows as well as many tokens of one. Scores, offsets, sums and O are f32; the probabilities are
// rounded to bf16 for the second product (each off by up to 2^-8 of itself, as much as a result in bf16 is).
#include <limits.h>

#include <algorithm>

#include "../../include/fv_sdpa_hip.h"
#include "packed.h"

namespace fv {
namespace {

constexpr int kRows = 128;             // of a workgroup, 32 a wave
constexpr float kLeast = 0x1p-149f;    // the weight of a seen key that vanished, where its value is not finite
constexpr float kLn2 = 0.69314718056f;

struct PackedAttnParams {
    PackedBatch b;
    PackedMask mask;
    const uint16_t *q, *k, *v;
    long q_stride, k_stride, v_stride;   // bytes between tokens
    void* out;                           // [tokens, heads, d]
    int out_is_bf16;
    float* lse;                          // [tokens, heads] or null
    int heads;
    PagedDiv group;                      // query heads that share a key head
    float sl2;                           // scale * log2(e)
    PagedPieces pieces;
    PackedRuns runs;
    int shares, chunk;                   // workgroups a walk, tiles of it that each takes
    // shares of walks longer than that: values, each normalised, and the base-2 logarithm of its sum: [shares][128 rows of every piece]
    float *part_o, *part_lse;
    long part_rows;
};

// 128 rows of one (sequence, key head), 32 a wave, over tiles of 64 keys that pass through LDS as in the dense kernels
// (attn_core.h): two buffers for K, two for V, so that a unit holds two workgroups, whose matrix and vector phases fall beside each other.
// A phase is one key tile: O += P V of the tile before and S = K Q^T with the next K and this V on their way in, the softmax, one barrier.
// (The softmax dealt out over the gaps between the products, as in the gradients: 4 % slower, the other workgroup's wave fills them better. Three
// buffers of 64 channels, loads a phase earlier: the same time. What bounds it: long walks of 128 channels the chip's power limit, 1.2 to
// 1.28 PFLOP/s; of 64 channels the softmax, 1.0 PFLOP/s; walks of a few tiles their ends, of 15 us for 8 tiles of 64 channels 1.6 to the piece,
// 0.7 to its loads, 1.8 for them and 1.9 from the last scores to the stores.)
// FIXED: a row's softmax offset stays at the largest score of the first tile (no row maximum and no rescale decision in the loop). Exact as
// long as nothing overflows or vanishes, which is checked before anything is stored: the sum of every row that sees a key of the
// walk within 2^-60 .. 2^100 and its values finite, or the workgroup makes the pass again with the running maximum and an eye on
// values that are not finite (returns false).
template <int D, bool FIXED, class Params>
FV_DEV bool packed_item_pass(const Params& p, const int wave, const int lane, const int block) {
    using G = TileGeo<D>;
    constexpr int kNO = D / 16, kTile = G::kTile, kIter = TileDma<4, D>::ITER, kUnits = kIter / 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
    lds_u8* smem = (lds_u8*)smem_raw;
    const int q4 = lane >> 4, i16 = lane & 15;
    const PackedSlot slot_at = packed_slot(p.runs, block, p.pieces.n.by * p.shares);
    if (slot_at.head < 0) return true;
    const int kvh = slot_at.head, share = paged_quot(slot_at.number, p.pieces.n);
    const int number = (share + 1) * p.pieces.n.by - 1 - slot_at.number;   // (a sequence's last rows, which see most, first)
    const PackedPiece piece = packed_piece<kRows>(p.pieces, p.b, p.group.by, number);
    const PackedSeq sq = piece.seq;
    const int rows = sq.count * p.group.by, row0 = piece.tile * kRows;
    if (row0 >= rows) return true;
    const int wrow = row0 + 32 * wave;
    const bool idle = wrow >= rows;   // (brings its part of the tiles and no more)
    bf16x8 qf[D / 32][2];             // (on their way before the walk is worked out: they come from the farthest)
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = min(wrow + 16 * g + i16, rows - 1), t = paged_quot(r, p.group);   // (past the last: the last again, not stored)
        const uint16_t* q = (const uint16_t*)((const uint8_t*)p.q + (long)(sq.start + t) * p.q_stride) + (kvh * p.group.by + r - t * p.group.by) * D + 8 * q4;
#pragma unroll
        for (int dk = 0; dk < D / 32; dk++) qf[dk][g] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(q + 32 * dk));
    }
    const PackedWalk w = packed_walk(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group));
    const int e0 = share * p.chunk, e1 = min(w.n, e0 + p.chunk);
    if (share > 0 && e0 >= e1) return true;
    const bool split = w.n > p.chunk;
    const float sl2 = p.sl2;

    unsigned koff[kIter], voff[kIter];
    packed_offsets<D>(koff, (unsigned)p.k_stride, wave, lane, [](int r) { return G::kswz(r); });
    packed_offsets<D>(voff, (unsigned)p.v_stride, wave, lane, [](int r) { return G::vswz(r); });
    const uint16_t *kbase = p.k + kvh * D, *vbase = p.v + kvh * D;
    const unsigned slot = (unsigned)(size_t)smem + wave * kIter * 1024;
    PackedRun krun(kbase, p.k_stride, sq, w, e0), vrun(vbase, p.v_stride, sq, w, e0);

    if (e0 < e1) {   // (with the queries: short walks are mostly this wait)
        const u32x4 kd = krun.rows(G::kRow), vd = vrun.rows(G::kRow);
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            packed_issue(kd, koff[2 * u], koff[2 * u + 1], slot + u * 2048);
            packed_issue(vd, voff[2 * u], voff[2 * u + 1], slot + 2 * kTile + u * 2048);
        }
    }

    // the wave's rows: the keys that all of them see, those of one of them a lane (row lane % 32; exchanged where a tile asks)
    PagedSight all_see = {0x7fffffff, 0, 0x7fffffff}, mine = {0, 0, 0};
    if (!idle) {
        all_see = packed_all(p.mask, sq, paged_quot(wrow, p.group), paged_quot(min(wrow + 32, rows) - 1, p.group));
        mine = packed_sight(p.mask, sq.pos0 + paged_quot(min(wrow + (lane & 31), rows - 1), p.group), sq.len);
    }
    const PackedWhole whole = packed_whole(w, all_see);
    const TileReadBases rb = tile_read_bases<D>(lane);
    auto kbuf = [&](int m) -> lds_u8* { return smem + (m & 1) * kTile; };
    auto vbuf = [&](int m) -> lds_u8* { return smem + (2 + (m & 1)) * kTile; };
    auto dst_row = [&](int r) {   // of the results
        const int t = paged_quot(r, p.group);
        return (size_t)(sq.start + t) * p.heads + kvh * p.group.by + (r - t * p.group.by);
    };
    auto part_row = [&](int r) { return (size_t)share * p.part_rows + (size_t)(kvh * p.pieces.n.by + number) * kRows + (r - row0); };
    f32x4 o[kNO][2], s_init[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    SoftmaxOffState st;
    st.init();
    ProbTile pb;

    // The second pass, a tile that some of the workgroup's rows see a part of: a value that is not finite belongs to the rows that see
    // it, whatever its weight, and a probability of zero does not keep it from the others. Such keys leave the V tile, and the rows
    // that see one add their share of it from memory. (The first pass ends in the check where there is such a value.)
    const PackedWhole wg_whole = packed_whole(w, packed_all(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group)));
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
            const int x = __builtin_ctzll(keys), key = w.key(e) + x;
            const uint16_t* vrow = (const uint16_t*)((const uint8_t*)vbase + (long)(sq.k0 + min(key, sq.len - 1)) * p.v_stride);
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
                const u32x2 v2 = *reinterpret_cast<const u32x2*>(vrow + 16 * db + 4 * q4);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = __builtin_bit_cast(float, i & 1 ? v2[i >> 1] & 0xffff0000u : v2[i >> 1] << 16);
#pragma unroll
                    for (int g = 0; g < 2; g++) o[db][g][i] += pj[g] == 0.f ? 0.f : pj[g] * v;
                }
            }
        }
        __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0), lgkmcnt(0)
        block_barrier();
    };
    auto mask_tile = [&](ScoreTile& s, int e) {
        if (whole.tile(e)) return;
        const unsigned m[3] = {(unsigned)mine.a, (unsigned)mine.lo, (unsigned)mine.hi};
        int both[3][2];   // the even rows of 16 lanes hold block 0's, the odd ones block 1's
#pragma unroll
        for (int x = 0; x < 3; x++) {
            const auto r = __builtin_amdgcn_permlane16_swap(m[x], m[x], false, false);
            both[x][0] = (int)r[0];
            both[x][1] = (int)r[1];
        }
        auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };   // bits of the first n of 4 keys
        const int key0 = w.key(e) + 4 * q4;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const int at = key0 + 16 * kb;
                const unsigned bits = below(both[0][g] - at) | (below(both[2][g] - at) & ~below(both[1][g] - at));
#pragma unroll
                for (int i = 0; i < 4; i++) s[kb][g][i] = (bits >> i) & 1 ? s[kb][g][i] : neg_inf();
            }
    };

#pragma unroll
    for (int db = 0; db < kNO; db++) o[db][0] = o[db][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (e0 < e1) {
#pragma unroll
        for (int dk = 0; dk < D / 32; dk++) asm volatile("" : "+v"(qf[dk][0]), "+v"(qf[dk][1]));   // (waited for here, not among the tile loads)
        wait_vmcnt<0>();
        block_barrier();
        constexpr int kAhead = 4;   // (three: 0.6 % slower, eight 1.2 %)
        krun.next(), vrun.next();
        u32x4 vd = vrun.rows(G::kRow), kd = krun.rows(G::kRow, e0 + 1 < e1);
        auto phase = [&](int m, auto first) {
            const int e = e0 + m;
            ScoreTile s;
            auto hook = [&](int i) {
                if constexpr (first()) i += kUnits;   // (the first values are there)
                if (i < kUnits) packed_issue(vd, voff[2 * i], voff[2 * i + 1], slot + (2 + (m & 1)) * kTile + i * 2048);
                else if (i < 2 * kUnits) packed_issue(kd, koff[2 * (i - kUnits)], koff[2 * (i - kUnits) + 1], slot + ((m + 1) & 1) * kTile + (i - kUnits) * 2048);
            };
            if (idle) {
#pragma unroll
                for (int i = 0; i < (first() ? 1 : 2) * kUnits; i++) hook(i);
            } else {
                __builtin_amdgcn_s_setprio(1);
                if constexpr (first()) mfma_phase<false, kAhead, D>(vbuf(0), kbuf(0), rb, pb, o, qf, s, s_init, hook);
                else mfma_phase<true, kAhead, D>(vbuf(m - 1), kbuf(m), rb, pb, o, qf, s, s_init, hook);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                mask_tile(s, e);
                if constexpr (first()) softmax_first_off<true>(s, st, s_init, sl2, pb);
                else if constexpr (FIXED) softmax_off_tile<true>(s, st, sl2, pb);
                else softmax_tile_off<true>(s, st, o, s_init, sl2, pb);
                asm volatile("" ::"v"(pb[0][0]), "v"(pb[0][1]), "v"(pb[1][0]), "v"(pb[1][1]), "v"(st.l_acc[0]), "v"(st.l_acc[1]));
            }
            if constexpr (!first()) vrun.next();
            krun.next();
            vd = vrun.rows(G::kRow), kd = krun.rows(G::kRow, e + 2 < e1);
            __builtin_amdgcn_sched_barrier(0);
            wait_vmcnt<0>();
            block_barrier();   // K(m + 1), V(m) resident; this phase's tiles read by every wave
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!FIXED) {
                if (!wg_whole.tile(e)) set_apart(m, e, pb, o);
            }
        };
        if (idle) {   // (defined for the second pass' shuffles and the votes)
#pragma unroll
            for (int t = 0; t < 2; t++) pb[t][0] = pb[t][1] = __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
        }
        phase(0, std::true_type{});
#pragma unroll 1
        for (int m = 1; m < e1 - e0; m++) phase(m, std::false_type{});
        if (!idle) pv_tile<D>(vbuf(e1 - e0 - 1), rb.v, pb, o);
    }

    if constexpr (FIXED) {
        // the lane's part of its rows' check; a row without a key in the walk has a sum of zero by right
        const int from = w.key(max(e0, w.ns)), to = w.key(max(e1 - 1, 0)) + kTileRows;
        const bool any = e0 < e1 && wrow + (lane & 31) < rows &&
                         ((e0 < w.ns && e0 * kTileRows < mine.a) || (e1 > w.ns && (max(mine.lo, from) < min(mine.hi, to) || from < mine.a)));
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
        // (of rows past the last nothing is stored; their values are the last's)
        const bool wave_ok = idle || __builtin_amdgcn_ballot_w64(!(fine && chk == 0.f)) == 0;
        // (the K buffer that neither the last P V nor the load past the walk's end uses is the one of this tile; all reads of it are behind a barrier)
        auto* votes = (__attribute__((address_space(3))) unsigned*)kbuf(e1 - e0 - 1);
        if (lane == 0) votes[wave] = wave_ok ? 0u : 1u;
        __builtin_amdgcn_s_waitcnt(0xC07F);
        block_barrier();
        const u32x4 v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(votes);
        const unsigned redo = (unsigned)__builtin_amdgcn_readfirstlane(v[0] | v[1] | v[2] | v[3]);
        if (redo != 0) {
            block_barrier();   // (a second pass loads over the votes)
            return false;
        }
    } else {
        block_barrier();   // (as the votes' one: the results pass through the V buffers, which every wave has read)
    }
    float inv[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const float l = quad_sum(st.l_acc[g]);
        inv[g] = l == 0.f ? 0.f : 1.f / l;
        const int r = wrow + 16 * g + i16;
        if (r >= rows || q4 != 0) continue;
        const float lse2 = l == 0.f ? neg_inf() : st.log2_offset<true>(g, sl2) + __log2f(l);
        if (split) p.part_lse[part_row(r)] = lse2;
        else if (p.lse) p.lse[dst_row(r)] = lse2 * kLn2;
    }
    if (!split && p.out_is_bf16) {   // (whole rows: 16 bytes a lane)
        if (idle) return true;
        bf16x4 y[kNO][2];
#pragma unroll
        for (int db = 0; db < kNO; db++)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                f32x4 x;
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = o[db][g][i] * inv[g];
                y[db][g] = __builtin_convertvector(x, bf16x4);
            }
        packed_store_rows<D>(smem + 2 * kTile + wave * (32 * G::kRow), y, lane,
                             [&](int r) -> uint16_t* { return wrow + r < rows ? (uint16_t*)p.out + dst_row(wrow + r) * D : nullptr; });
        return true;
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = wrow + 16 * g + i16;
        if (r >= rows) continue;
        float* to = split ? p.part_o + part_row(r) * D : (float*)p.out + dst_row(r) * D;
#pragma unroll
        for (int db = 0; db < kNO; db++) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = o[db][g][i] * inv[g];
            *reinterpret_cast<f32x4*>(to + 16 * db + 4 * q4) = x;
        }
    }
    return true;
}

// The kernel's arguments read again from their segment, of which PackedAttnParams is the whole, and the lane counted anew, so that the
// second pass keeps nothing of the first in registers.
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_attn_kernel(const PackedAttnParams p) {
    int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = blockIdx.x;
    if (packed_item_pass<D, true>(p, wave, threadIdx.x & 63, block)) return;
    using ConstParams = const __attribute__((address_space(4))) PackedAttnParams;
    ConstParams* again = (ConstParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(again));
    int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane), "+s"(wave), "+s"(block));
    packed_item_pass<D, false>(*again, wave, lane, block);
}

// The shares of a split walk joined: out = sum_c w_c O_c / sum_c w_c, w_c = 2^(lse_c - max lse); D / 4 threads a row. Rows whose walk
// one workgroup made have their result already.
template <int D>
__global__ __launch_bounds__(256) void packed_join_kernel(const PackedAttnParams p) {
    constexpr int kPer = D / 4, kJoin = 256 / kPer, kPerPiece = kRows / kJoin;
    const int c = threadIdx.x % kPer, slot = threadIdx.x / kPer;
    const int item = blockIdx.x / kPerPiece, kvh = paged_quot(item, p.pieces.n), number = item - kvh * p.pieces.n.by;
    const PackedPiece piece = packed_piece<kRows>(p.pieces, p.b, p.group.by, number);
    const PackedSeq sq = piece.seq;
    const int rows = sq.count * p.group.by, row0 = piece.tile * kRows;
    if (row0 >= rows) return;
    const PackedWalk w = packed_walk(p.mask, sq, paged_quot(row0, p.group), paged_quot(min(row0 + kRows, rows) - 1, p.group));
    const int in = (int)(blockIdx.x % kPerPiece) * kJoin + slot, r = row0 + in;
    if (w.n <= p.chunk || r >= rows) return;
    const int shares = (w.n + p.chunk - 1) / p.chunk;
    const size_t first = (size_t)item * kRows + in;
    float top = neg_inf(), total = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < shares; s += 4) {
        float lse[4];
        f32x4 x[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const size_t at = (size_t)min(s + u, shares - 1) * p.part_rows + first;
            lse[u] = p.part_lse[at];
            x[u] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + 4 * c);
        }
        float m = top;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (s + u >= shares) lse[u] = neg_inf();
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
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int t = paged_quot(r, p.group);
    const size_t dst = (size_t)(sq.start + t) * p.heads + kvh * p.group.by + (r - t * p.group.by);
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] *= inv;
    if (p.out_is_bf16) *reinterpret_cast<bf16x4*>((uint16_t*)p.out + dst * D + 4 * c) = __builtin_convertvector(acc, bf16x4);
    else *reinterpret_cast<f32x4*>((float*)p.out + dst * D + 4 * c) = acc;
    if (c == 0 && p.lse) p.lse[dst] = total == 0.f ? neg_inf() : (top + __log2f(total)) * kLn2;
}

// How a call is cut: tiles of a walk that a workgroup takes, workgroups a walk.
struct PackedCut {
    PagedPieces pieces;
    size_t chunk, shares;
    size_t rows(size_t kv_heads) const { return kv_heads * (size_t)pieces.n.by * kRows; }
    size_t bytes(size_t kv_heads, size_t d) const { return shares > 1 ? (shares * rows(kv_heads) * (d + 1) * 4 + 255) / 256 * 256 : 0; }
};
constexpr size_t kMostShares = (size_t)1 << 30;   // bytes of a call's shares: past it its walks are cut less
PackedCut packed_cut(const PackedCall& c) {
    const size_t group = c.heads / c.kv_heads, units = (size_t)fv_compute_units(), slots = (c.d == 64 ? 3 : 2) * units;
    PackedCut cut;
    cut.pieces = paged_pieces(kRows, c.seqs, c.tokens, c.max_q, group);
    const size_t steps = fv_packed_key_steps(c, kRows), items = c.kv_heads * (size_t)cut.pieces.n.by;
    // (ragged: one number a sequence may be unused)
    const size_t held = cut.pieces.tiles.by ? items : std::max<size_t>(c.kv_heads * (c.tokens * group / kRows + 1), items / 2);
    size_t shares = held < slots ? std::min(slots / held, std::max<size_t>(steps / 4, 1)) : 1;
    shares = std::min(shares, std::max<size_t>(kMostShares / std::max<size_t>(items * kRows * (c.d + 1) * 4, 1), 1));
    cut.chunk = (steps + shares - 1) / shares;
    cut.shares = (steps + cut.chunk - 1) / cut.chunk;
    return cut;
}

}  // namespace
}  // namespace fv

size_t fv_packed_key_steps(const PackedCall& c, size_t rows) {
    size_t steps = (c.max_k + fv::kTileRows - 1) / fv::kTileRows;
    if (c.causal && c.window > 0) {   // the first token's window and the blocks to the last token's, a step more (they begin anywhere in one); the sink
        const size_t group = c.heads / c.kv_heads, apart = (rows + group - 2) / group, blocks = c.window + (apart + c.block_tokens - 1) / c.block_tokens;
        const size_t far = (size_t)1 << 31;
        const size_t band = blocks < far / c.block_tokens ? blocks * c.block_tokens : far, keep = c.sink < far / c.block_tokens ? c.sink * c.block_tokens : far;
        steps = std::min(steps, (band + fv::kTileRows - 1) / fv::kTileRows + 1 + (keep + fv::kTileRows - 1) / fv::kTileRows);
    }
    return std::max<size_t>(steps, 1);
}

static bool mask_fits(const PackedCall& c) { return std::max({c.block_tokens, c.window, c.sink}) <= (size_t)INT_MAX / 2; }
bool fv_packed_sizes(const PackedCall& c) {
    return c.kv_heads > 0 && c.heads >= c.kv_heads && c.heads % c.kv_heads == 0 && c.heads <= 65535 && (c.d == 64 || c.d == 128) && c.seqs > 0 &&
           c.seqs <= kMostSeqs && c.tokens <= kMostRows && c.k_tokens <= kMostRows && c.tokens * (c.heads / c.kv_heads) <= (size_t)INT_MAX / 2 &&
           (!c.causal || (c.block_tokens > 0 && mask_fits(c)));
}
fv::PackedMask fv_packed_mask(const PackedCall& c) {
    return {c.causal != 0, fv::paged_div(c.causal ? c.block_tokens : 1), c.causal ? (int)c.window : 0, c.causal ? (int)c.sink : 0};
}
int fv_packed_args(const char* who, const PackedCall& c, const PackedOperand* x, size_t operands, const void* workspace) {
    auto say = [who](const char* why, bool decline) {
        char buf[200];
        snprintf(buf, sizeof buf, "%s: %s", who, why);
        return decline ? fv_decline(buf) : fv_invalid(buf);
    };
    if (!c.q_start || !c.k_start) return say("null operand", false);
    if (c.heads == 0 || c.kv_heads == 0 || c.heads % c.kv_heads != 0) return say("query heads must be a multiple of the key heads", false);
    if (c.d != 64 && c.d != 128) return say("head dim must be 64 or 128", true);
    if (c.heads > 65535) return say("too many heads", true);
    if (c.seqs > kMostSeqs || c.tokens > kMostRows || c.k_tokens > kMostRows || c.tokens * (c.heads / c.kv_heads) > (size_t)INT_MAX / 2)
        return say("too many sequences or rows for one launch", true);
    if (!(c.scale >= 1e-30f) || !(c.scale <= 1e30f)) return say("scale must lie within 1e-30 and 1e30", true);   // (the gradients' lse / scale is a number)
    if (c.causal && c.block_tokens == 0) return say("block_tokens must be positive", false);
    if (c.causal && !mask_fits(c)) return say("mask too large", true);
    for (size_t i = 0; i < operands; i++) {
        if (!x[i].at) return say("null operand", false);
        if (((uintptr_t)x[i].at & 15) != 0) return say("operands must be 16-byte aligned", false);
        if (x[i].stride < x[i].heads * c.d) return say("tokens overlap (a stride below heads * d)", false);
        // (a tile's 64 rows lie within 32 bits of bytes)
        if (x[i].stride % 8 != 0 || x[i].stride > (size_t)1 << 24) return say("strides must be multiples of 8 elements, 2^24 at most", true);
    }
    if (((uintptr_t)workspace & 255) != 0) return say("the workspace must be 256-byte aligned", false);
    return FV_OK;
}

extern "C" {

size_t fv_packed_attention_workspace_bytes(size_t heads, size_t kv_heads, size_t d, size_t seqs, size_t q_tokens, size_t k_tokens, size_t max_q,
                                           size_t max_k, int causal, size_t block_tokens, size_t window, size_t sink) {
    const PackedCall c = {heads, kv_heads, d, seqs, q_tokens, k_tokens, std::min(max_q, q_tokens), std::min(max_k, k_tokens), nullptr, nullptr, 1.f, causal,
                          block_tokens, window, sink};
    return fv_packed_sizes(c) && c.max_q > 0 ? fv::packed_cut(c).bytes(kv_heads, d) : 0;
}

int fv_packed_attention(const uint16_t* q, size_t q_stride, const uint16_t* k, size_t k_stride, const uint16_t* v, size_t v_stride, void* out,
                        int out_is_bf16, float* lse, size_t heads, size_t kv_heads, size_t d, const int32_t* q_start, const int32_t* k_start,
                        size_t seqs, size_t q_tokens, size_t k_tokens, size_t max_q, size_t max_k, float scale, int causal, size_t block_tokens,
                        size_t window, size_t sink, void* workspace, size_t workspace_bytes, void* stream) {
    if (seqs == 0 || q_tokens == 0 || max_q == 0) return FV_OK;   // (empty arrays may have no address)
    const PackedCall c = {heads, kv_heads, d, seqs, q_tokens, k_tokens, std::min(max_q, q_tokens), std::min(max_k, k_tokens), q_start, k_start, scale,
                          causal, block_tokens, window, sink};
    const bool keys = k_tokens > 0;   // (without any, no address is followed)
    const PackedOperand x[] = {{q, q_stride, heads}, {out, heads * d, heads}, {keys ? k : q, keys ? k_stride : q_stride, keys ? kv_heads : heads},
                               {keys ? v : q, keys ? v_stride : q_stride, keys ? kv_heads : heads}};
    const int rc = fv_packed_args("packed attention", c, x, 4, workspace);
    if (rc != FV_OK) return rc;
    fv::PackedCut cut = fv::packed_cut(c);
    if (cut.bytes(kv_heads, d) > 0 && (!workspace || workspace_bytes < cut.bytes(kv_heads, d))) cut.chunk *= cut.shares, cut.shares = 1;
    fv::PackedAttnParams p;
    p.b = {q_start, k_start, (int)seqs, (int)q_tokens, (int)k_tokens, (int)c.max_q, (int)c.max_k};
    p.mask = fv_packed_mask(c);
    p.q = q, p.k = k, p.v = v;
    p.q_stride = (long)q_stride * 2, p.k_stride = (long)k_stride * 2, p.v_stride = (long)v_stride * 2;
    p.out = out, p.out_is_bf16 = out_is_bf16 != 0, p.lse = lse;
    p.heads = (int)heads, p.group = fv::paged_div(heads / kv_heads);
    p.sl2 = (float)((double)scale * 1.4426950408889634);
    p.pieces = cut.pieces, p.chunk = (int)cut.chunk;
    const size_t items = kv_heads * (size_t)cut.pieces.n.by;
    constexpr size_t kMost = (size_t)1 << 24;   // (a launch holds fewer than 2^32 work-items)
    const size_t join_blocks = items * fv::kRows / (1024 / d);
    if (items * cut.shares >= kMost / 2 || (cut.shares > 1 && join_blocks >= kMost)) return fv_decline("packed attention: too large for one launch");
    p.runs = fv::packed_runs(kv_heads, causal != 0), p.shares = (int)cut.shares;
    p.part_rows = (long)cut.rows(kv_heads);
    p.part_o = (float*)workspace, p.part_lse = p.part_o + cut.shares * cut.rows(kv_heads) * d;
    hipStream_t st = (hipStream_t)stream;
    fv::paged_pick(d == 128, [&](auto d128) {
        constexpr int D = d128() ? 128 : 64;
        hipLaunchKernelGGL((fv::packed_attn_kernel<D>), dim3((unsigned)fv::packed_blocks(p.runs, (size_t)cut.pieces.n.by * cut.shares)), dim3(256), 4 * fv::TileGeo<D>::kTile, st, p);
        if (cut.shares > 1) hipLaunchKernelGGL((fv::packed_join_kernel<D>), dim3((unsigned)join_blocks), dim3(256), 0, st, p);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "packed_attention");
}

}  // extern "C"
