// Packed sequences: the tokens of sequences of different lengths one behind the other in [tokens, heads, d] tensors, queries and keys
// with starts of their own. What the kernels of the attention (packed_attn.hip) and of its gradients (packed_back.hip) share.
#pragma once
#include <utility>

#include "attn_core.h"
#include "fv_internal.h"
#include "paged.h"

namespace fv {

// Sequence s: rows q_start[s] .. q_start[s + 1] of the queries, k_start[s] .. k_start[s + 1] of the keys. Device memory that the host does
// not see: bounded here to the tensors' rows.
struct PackedBatch {
    const int* q_start;
    const int* k_start;
    int seqs, tokens, k_tokens, max_q, max_k;   // (a sequence's rows and keys past the bounds that the launch is sized by are left out)
};
// The keys' side alone, for numbering pieces of keys.
struct PackedKeys {
    const int* q_start;
    int seqs, tokens;
};

struct PackedSeq {
    int start, count;   // first row, rows
    int k0, len;        // first key, keys
    int pos0;           // position of the first row among the keys: the last row of the whole sequence is at its last key, also where max_q or max_k
};                      // leave some out; negative where rows are more than keys
// Of the rows [q0, q1) and the keys [k0, k1) those within the bounds.
template <class Batch>
FV_DEV PackedSeq packed_within(const Batch& b, int q0, int q1, int k0, int k1) {
    return {q0, min(q1 - q0, b.max_q), k0, min(k1 - k0, b.max_k), (k1 - k0) - (q1 - q0)};
}
template <class Batch>
FV_DEV PackedSeq packed_seq(const Batch& b, int s) {
    const int q0 = min(max(b.q_start[s], 0), b.tokens), k0 = min(max(b.k_start[s], 0), b.k_tokens);
    return packed_within(b, q0, min(max(b.q_start[s + 1], q0), b.tokens), k0, min(max(b.k_start[s + 1], k0), b.k_tokens));
}

// The piece of a number and its sequence (of a whole wave). Up to 63 sequences: the starts come with one load of the wave, from which both the search and
// the sequence are taken.
struct PackedPiece {
    PackedSeq seq;
    int tile;   // (one that the sequence does not have: of an unused number)
};
template <int R, class Pieces, class Batch>
FV_DEV PackedPiece packed_piece(const Pieces& x, const Batch& b, int group, int number) {
    if (x.tiles.by || b.seqs > 63) {
        const PagedPiece at = paged_piece<R>(x, b, group, number);
        return {packed_seq(b, at.seq), at.tile};
    }
    const int lane = threadIdx.x & 63, row = b.q_start[min(lane, b.seqs)], key = b.k_start[min(lane, b.seqs)];
    const long first = ((long)min(max(row, 0), b.tokens) * group + (long)(R - 1) * lane) / R;
    const int seq = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < b.seqs && first <= number)), 1) - 1;
    const int q0 = min(max(__builtin_amdgcn_readlane(row, seq), 0), b.tokens), k0 = min(max(__builtin_amdgcn_readlane(key, seq), 0), b.k_tokens);
    const int q1 = min(max(__builtin_amdgcn_readlane(row, seq + 1), q0), b.tokens), k1 = min(max(__builtin_amdgcn_readlane(key, seq + 1), k0), b.k_tokens);
    const long tile = number - ((long)q0 * group + (long)(R - 1) * seq) / R;
    constexpr int kNone = 0x7fffffff / R;
    return {packed_within(b, q0, q1, k0, k1), tile < 0 || tile > kNone ? kNone : (int)tile};
}

// f(0), f(1), .., f(N - 1) with the numbers as types (loops that the compiler does not unroll in time).
template <class F, int... I>
FV_DEV void static_for_each(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
FV_DEV void static_for(F&& f) {
    static_for_each(f, std::make_integer_sequence<int, N>{});
}

// The mask: without `causal` every row sees every key of its sequence; with it as in paged_sight.
struct PackedMask {
    int causal;
    PagedDiv block_tokens;
    int window, sink;
};
template <class Mask>
FV_DEV PagedSight packed_sight(const Mask& m, int pos, int len) {
    return m.causal ? paged_sight(m, pos, len) : PagedSight{0, 0, len};
}
template <class Mask>
FV_DEV PagedSight packed_all(const Mask& m, const PackedSeq& s, int t0, int t1) {   // what the tokens t0 .. t1 all see
    const PagedSight f = packed_sight(m, s.pos0 + t0, s.len), l = packed_sight(m, s.pos0 + t1, s.len);
    return {f.a, l.lo, f.hi};
}

// The walk of a tile of rows (tokens t0 .. t1 of the sequence) over tiles of 64 keys: the first ns hold the sink, then from tile b0.
struct PackedWalk {
    int ns, b0, n;
    PagedSight any;   // the keys that some row sees
    FV_DEV int key(int e) const { return (e < ns ? e : b0 + e - ns) * kTileRows; }
    // the tiles of the walk before key 64 t
    FV_DEV int before(int t) const { return min(t, ns) + min(max(t - b0, 0), n - ns); }
};
template <class Mask>
FV_DEV PackedWalk packed_walk(const Mask& m, const PackedSeq& s, int t0, int t1) {
    PackedWalk w;
    const PagedSight l = packed_sight(m, s.pos0 + t1, s.len);
    w.any = {l.a, packed_sight(m, max(s.pos0 + t0, 0), s.len).lo, l.hi};
    w.ns = (w.any.a + kTileRows - 1) / kTileRows;
    w.b0 = max(w.any.lo / kTileRows, w.ns);
    w.n = w.ns + max(0, (w.any.hi + kTileRows - 1) / kTileRows - w.b0);
    return w;
}
// The tiles of the walk that rows which all see `all` see whole: those before `a` and [b, c).
struct PackedWhole {
    int a, b, c;
    FV_DEV bool tile(int e) const { return e < a || (e >= b && e < c); }
};
FV_DEV PackedWhole packed_whole(const PackedWalk& w, const PagedSight& all) {
    return {w.before(all.a / kTileRows), all.a >= all.lo ? 0 : w.before((all.lo + kTileRows - 1) / kTileRows), w.before(all.hi / kTileRows)};
}

// Workgroups to pieces: 2^xcds XCDs take the pieces of a run of whole key heads, in turn, so that an L2 holds few heads' tensors. Under a causal mask the
// heads' pieces follow each other by number, so that the longest walks of all come first (one clip of 7 frames, 12 heads, three a run: 13 % over even
// shares of the work instead of 36 %); where walks are alike, head by head (two clips, 12 heads, forward: 727 us, by number 751).
struct PackedRuns {
    PagedDiv heads;   // of a run
    int xcds, by_head;
};
struct PackedSlot {
    int head, number;   // of the key head's pieces; head < 0: none
};
template <class Runs>
FV_DEV PackedSlot packed_slot(const Runs& x, int block, int numbers) {
    const int in_run = ((block >> 3) << x.xcds) + (block & ((1 << x.xcds) - 1)), first = ((block & 7) >> x.xcds) * x.heads.by;
    if (numbers <= 0) return {-1, 0};
    const int a = x.by_head ? in_run / numbers : paged_quot(in_run, x.heads), b = in_run - a * (x.by_head ? numbers : x.heads.by);
    const int head = x.by_head ? a : b, number = x.by_head ? b : a;
    return {head < x.heads.by && number < numbers ? first + head : -1, number};
}
inline PackedRuns packed_runs(size_t kv_heads, bool causal) {
    const int xcds = kv_heads % 8 == 0 ? 0 : kv_heads % 4 == 0 ? 1 : kv_heads % 2 == 0 ? 2 : 3;
    return {paged_div(kv_heads >> (3 - xcds)), xcds, causal ? 0 : 1};
}
inline size_t packed_blocks(const PackedRuns& x, size_t numbers) {
    return (((size_t)x.heads.by * numbers + ((size_t)1 << x.xcds) - 1) >> x.xcds) * 8;
}

// Per-lane source offsets of a wave's part of a 64-row tile whose rows lie `stride` bytes apart (ITER loads a wave of four, in the LDS
// layout of attn_core.h). Second loads of a pair less the 1 KB that their immediate offset adds.
template <int D, int ITER, class Swz>
FV_DEV void packed_offsets(unsigned (&off)[ITER], unsigned stride, int wave, int lane, Swz&& swz) {
    using G = TileGeo<D>;
#pragma unroll
    for (int it = 0; it < ITER; it++) {
        const int r = (wave * ITER + it) * G::kRowsPerDma + lane / G::kChunks, c = lane % G::kChunks;
        off[it] = (unsigned)r * stride + ((unsigned)(c ^ swz(r)) << 4) - (unsigned)(it & 1) * 1024u;
    }
}
// Rows [first, first + count) of a head whose rows lie `stride` bytes apart, count <= 64, as a descriptor: rows behind them are zeros.
FV_DEV u32x4 packed_rows(const uint16_t* base, long first, long stride, int count, int row_bytes) {
    return plane_descriptor((const uint8_t*)base + first * stride, count > 0 ? (unsigned)((long)(count - 1) * stride) + (unsigned)row_bytes : 0u);
}
// The tiles of a walk over K or V, one after the other: where a tile lies goes on by one product that is made once.
struct PackedRun {
    const uint8_t* at;
    long step, jump;   // to the next tile; from the sink's last to the band's first, besides
    unsigned stride;
    int left, gap;     // keys of the sequence from the tile's first; keys between the sink's tiles and the band's
    int e, ns;
    FV_DEV PackedRun(const uint16_t* base, long stride_, const PackedSeq& s, const PackedWalk& w, int e_) {
        e = e_, ns = w.ns, stride = (unsigned)stride_;
        const int key = w.key(e);
        at = (const uint8_t*)base + (s.k0 + key) * stride_, left = s.len - key;
        step = kTileRows * stride_, gap = (w.b0 - w.ns) * kTileRows, jump = gap * stride_;
    }
    FV_DEV u32x4 rows(int row_bytes, bool any = true) const {   // (none: zeros)
        return plane_descriptor(at, any && left > 0 ? (unsigned)(min(left, kTileRows) - 1) * stride + (unsigned)row_bytes : 0u);
    }
    FV_DEV void next() {
        e++;
        at += step, left -= kTileRows;
        if (e == ns) at += jump, left -= gap;
    }
};
// Two loads of a wave into LDS at `lds` (wave-uniform).
FV_DEV void packed_issue(const u32x4& rows, unsigned o0, unsigned o1, unsigned lds) {
    const unsigned m0 = (unsigned)__builtin_amdgcn_readfirstlane((int)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                 "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 lds"
                 :: "s"(m0), "v"(o0), "v"(o1), "s"(rows) : "memory");
}

// A wave's 32 rows in bf16, x[db][g] its lanes' channels 16 db + 4 q4 .. + 3 of row 16 g + i16: through 32 x 2D bytes of LDS of the wave's own, scattered
// 8-byte pieces in, whole rows out, 16 bytes a lane. dst(row): where a row lies, or null.
template <int D, class Dst>
FV_DEV void packed_store_rows(lds_u8* my, const bf16x4 (&x)[D / 16][2], int lane, Dst&& dst) {
    constexpr int kRowB = 2 * D, kCh = kRowB / 16, kRowsPer = 64 / kCh;
    const int q4 = lane >> 4, i16 = lane & 15;
#pragma unroll
    for (int db = 0; db < D / 16; db++)
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int ch = (2 * db + (q4 >> 1)) ^ (i16 & (kCh - 1));
            *reinterpret_cast<__attribute__((address_space(3))) bf16x4*>(my + (16 * g + i16) * kRowB + (ch << 4) + 8 * (q4 & 1)) = x[db][g];
        }
    // (writes and reads of one wave complete in order; the compiler waits for the reads' data)
    const int c = lane % kCh;
    u32x4 v[32 / kRowsPer];
#pragma unroll
    for (int i = 0; i < 32 / kRowsPer; i++) {
        const int r = i * kRowsPer + lane / kCh;
        v[i] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(my + r * kRowB + ((c ^ (r & (kCh - 1))) << 4));
    }
#pragma unroll
    for (int i = 0; i < 32 / kRowsPer; i++) {
        uint16_t* to = dst(i * kRowsPer + lane / kCh);
        if (to) global_store<u32x4>(to + 8 * c, v[i]);
    }
}

}  // namespace fv

// What the entries check alike; FV_OK, or what they return. Operands: bf16 bits [tokens, heads, d], tokens a stride apart.
struct PackedOperand {
    const void* at;
    size_t stride, heads;
};
struct PackedCall {
    size_t heads, kv_heads, d, seqs, tokens, k_tokens, max_q, max_k;
    const int32_t *q_start, *k_start;
    float scale;
    int causal;
    size_t block_tokens, window, sink;
};
int fv_packed_args(const char* who, const PackedCall& c, const PackedOperand* x, size_t operands, const void* workspace);
fv::PackedMask fv_packed_mask(const PackedCall& c);
// Numbers whose workspace is asked for, within what the entries take.
bool fv_packed_sizes(const PackedCall& c);
// Tiles of 64 keys that the walk of a piece of `rows` rows may have, by the call's bounds.
size_t fv_packed_key_steps(const PackedCall& c, size_t rows);
