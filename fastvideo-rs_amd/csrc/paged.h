// The paged KV cache: where a token of a sequence lies, and what a query sees of its sequence. Shared by the kernels that
// write and read the pages (paged_kv.hip) and the attention over them (paged_attn.hip).
#pragma once
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
