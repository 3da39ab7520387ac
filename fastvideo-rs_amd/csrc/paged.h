// Ragged batches: how a launch numbers their rows, what a query sees of its sequence, and, of the paged KV cache, where a token lies.
// Shared by the kernels that write and read the pages (paged_kv.hip), the attention over them (paged_attn.hip) and that over packed
// sequences and its gradients (packed.h).
#pragma once
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "fv_common.h"

namespace fv {

// Pages [pages, kv_heads, 1 << lg, d] of bf16, or (ks, vs not null) of 4 bits: codes [.., d / 2] (e2m1, channel 2i in the low
// half of byte i) and scales [.., d / 32] (e8m0: 2^(byte - 127), 255: not a number).
struct PagedPool {
    void* k;
    void* v;
    uint8_t* ks;
    uint8_t* vs;
    int pages, lg, kv_heads;
};

// The batch: sequence s has lens[s] tokens in the cache, of which the last ones are the rows q_start[s] .. q_start[s + 1] of
// the call's ragged tensors; token j lies in slot j % page_tokens of page table[s][j / page_tokens]. All of it is device
// memory that the host does not see, so every use is bounded here: rows to `tokens`, lengths to `max_len` (no more than the
// table's columns hold), page numbers by the readers.
struct PagedBatch {
    const int* q_start;
    const int* lens;
    const int* table;
    long table_stride;
    int seqs, tokens, max_len;
};

struct PagedSeq {
    int start, count, len;   // first row, rows, tokens in the cache
    int behind;              // the row behind its last token, which the call's tensors need not have
    FV_DEV int first_pos() const { return pos_of(len); }   // of row `start`; negative where there are more rows than tokens
    FV_DEV int pos_of(int length) const { return length - (behind - start); }
};
template <class Batch>   // (PagedBatch, or the same struct read through another address space)
FV_DEV PagedSeq paged_seq(const Batch& b, int s) {
    PagedSeq q;
    q.start = min(max(b.q_start[s], 0), b.tokens);
    q.behind = max(b.q_start[s + 1], q.start);
    q.count = min(q.behind, b.tokens) - q.start;
    q.len = min(max(b.lens[s], 0), b.max_len);
    return q;
}

// Division of a number below 2^31 by one that the host knows, as a product and a shift: with 2^l >= by, mul = 2^(31 + l) / by rounded up is
// too large by less than 1, so n mul / 2^(31 + l) by less than 1 / by. (The compiler's own takes 20 instructions and waits for a
// reciprocal; a workgroup makes ten of them before its first load.)
struct PagedDiv {
    unsigned mul;
    int shift, by;
};
template <class Div>
FV_DEV int paged_quot(int n, const Div& d) { return (int)(((unsigned long long)(unsigned)n * d.mul) >> d.shift); }
inline PagedDiv paged_div(size_t by) {   // below 2^31 (0: never used)
    if (by == 0) return {0, 0, 0};
    int l = 0;
    while (((size_t)1 << l) < by) l++;
    return {(unsigned)((1ull << (31 + l)) / by + 1), 31 + l, (int)by};
}

// Pieces of up to R rows of the (token, head of the group) rows of a batch, for one key head. Where the sequences are as long as
// the longest, piece t of sequence s is number s tiles + t. Where they are not (tiles 0), it is number first(s) + t with
// first(s) = (group q_start[s] + (R - 1) s) / R, which leaves each its ceil(rows / R) numbers and no more than one for each sequence
// unused, whatever the longest is. (A prompt of 8192 tokens among 255 single ones: 6.8 ms with the longest's pieces for all.)
struct PagedPieces {
    PagedDiv n, tiles;          // numbers, of a sequence
};
struct PagedPiece {
    int seq, tile;              // (of an unused number: a tile that the sequence does not have, R tile below 2^31)
};
template <int R, class Pieces, class Batch>
FV_DEV long paged_first_piece(const Pieces& x, const Batch& b, int group, int seq) {
    return x.tiles.by ? (long)seq * x.tiles.by : ((long)min(max(b.q_start[seq], 0), b.tokens) * group + (long)(R - 1) * seq) / R;
}
template <int R, class Pieces, class Batch>
FV_DEV PagedPiece paged_piece(const Pieces& x, const Batch& b, int group, int number) {   // (of a whole wave)
    if (x.tiles.by) {
        const int seq = paged_quot(number, x.tiles);
        return {seq, number - seq * x.tiles.by};
    }
    const int lane = threadIdx.x & 63;
    int seq = 0, n = b.seqs;    // the last of sequences seq .. seq + n - 1 whose first piece is no later: 64 of them at a time
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const bool le = at < n && paged_first_piece<R>(x, b, group, seq + min(at, n - 1)) <= number;
        const int k = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(le)), 1) - 1;
        seq += k * step;
        n = min(step, n - k * step);
    }
    const long tile = number - paged_first_piece<R>(x, b, group, seq);   // (negative: of rows before the first sequence)
    constexpr int kNone = 0x7fffffff / R;
    return {seq, tile < 0 || tile > kNone ? kNone : (int)tile};
}

inline PagedPieces paged_pieces(size_t r, size_t seqs, size_t tokens, size_t max_q, size_t group) {
    const size_t tiles = (max_q * group + r - 1) / r, like = seqs * tiles, ragged = (tokens * group + (r - 1) * seqs) / r;
    const size_t most = INT_MAX;   // (past it no launch holds them)
    return like <= ragged ? PagedPieces{paged_div(std::min(like, most)), paged_div(std::min(tiles, most))}
                          : PagedPieces{paged_div(std::min(ragged, most)), paged_div(0)};
}

// The keys that a row at position p of a sequence of `len` tokens sees: [0, a) and [lo, hi), a <= hi.
struct PagedSight {
    int a, lo, hi;
    // bit j: key k + j, j < 8. (Bits and selects: the comparisons key by key under divergent branches were compiled into
    // code that lost the stores of -inf.)
    FV_DEV unsigned eight(int k) const {
        return below(a - k) | (below(hi - k) & ~below(lo - k));
    }
    static FV_DEV unsigned below(int n) { return (1u << min(max(n, 0), 8)) - 1u; }
    FV_DEV bool one(int k) const { return k < a || (k >= lo && k < hi); }
};
template <class Params>
FV_DEV PagedSight paged_sight(const Params& p, int pos, int len) {
    if (pos < 0) return {0, 0, 0};
    const int bt = p.block_tokens.by, block = paged_quot(pos, p.block_tokens);
    const long hi = (long)(block + 1) * bt, sink = (long)p.sink * bt;
    PagedSight s;
    s.hi = (int)min(hi, (long)len);
    s.lo = p.window > 0 ? max(0, block - p.window + 1) * bt : 0;
    s.a = (int)min(sink, (long)s.hi);
    return s;
}

// Bytes of one row of one head: values, scales.
template <int D, bool FOUR>
struct PagedGeo {
    static constexpr int kRow = FOUR ? D / 2 : 2 * D;
    static constexpr int kScales = D / 32;
};

FV_DEV float e8m0_scale(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

// One byte of `w` (two 4-bit codes) times the scale, as two bf16: exact, the conversion of the instruction set.
template <int BYTE>
FV_DEV unsigned fp4_pair(unsigned w, float scale) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE));
}
// Eight codes to eight bf16 in four words.
FV_DEV u32x4 fp4_eight(unsigned w, float scale) {
    return u32x4{fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale)};
}

// NaN where one of the two bf16 of a word is not finite, else `x`: for testing many.
FV_DEV float not_finite(unsigned w, float x) {
    return __builtin_fmaf(__builtin_bit_cast(float, w & 0xffff0000u), 0.f, __builtin_fmaf(__builtin_bit_cast(float, w << 16), 0.f, x));
}

// f(std::true_type) or f(std::false_type): host values as template arguments.
template <class F>
inline void paged_pick(bool v, F&& f) {
    if (v) f(std::true_type{});
    else f(std::false_type{});
}

}  // namespace fv

constexpr size_t kMostSeqs = (size_t)1 << 24, kMostRows = (size_t)1 << 26;   // of a call
int fv_paged_args(const char* who, const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, size_t pages,
                  size_t page_tokens, size_t kv_heads, size_t d, const int32_t* q_start, const int32_t* lens, const int32_t* table,
                  size_t table_stride, size_t table_pages, size_t seqs, size_t tokens, const size_t* max_len, fv::PagedPool* pool,
                  fv::PagedBatch* b);
