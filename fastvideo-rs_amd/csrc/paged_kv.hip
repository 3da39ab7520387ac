// Writing and reading the pages of a paged KV cache (declarations: include/fv_sdpa_hip.h): new tokens of a ragged batch go
// in with the rotation of their positions applied on the way, as bf16 or as 4-bit codes, and come out again as rows.
//
// Both are HBM-bound scans: a thread moves 8 channels of one head of a token in one 16-byte piece (two for f32), a workgroup
// takes 256 such pieces of one token, so that the sequence, the page and the slot are scalars, computed once, and every load
// and store of a wave is a run of neighbouring pieces.
#include <limits.h>
#include <stdio.h>

#include "../../include/fv_sdpa_hip.h"
#include "fv_common.h"
#include "fv_internal.h"
#include "paged.h"

namespace fv {
namespace {

struct AppendParams {
    PagedPool pool;
    PagedBatch b;
    const void* k;
    const void* v;
    const void* q;
    uint16_t* q_out;
    long k_stride, v_stride, q_stride;   // elements between tokens
    const float* cos_t;                  // [rope_rows, d], or null: no rotation
    const float* sin_t;
    const int* rope_at;                  // row of each token, or null: its position
    int rope_rows, heads;
};

// The sequence that row t belongs to: the last s with q_start[s] <= t. One token a sequence is looked up at once.
FV_DEV int paged_seq_of(const PagedBatch& b, int t) {
    if (t < b.seqs && b.q_start[t] <= t && b.q_start[t + 1] > t) return t;
    int lo = 0, hi = b.seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Where row t of the batch lies in the cache: its position (-1: in no sequence, or before one's first token), page (-1 where the
// table or the pool has no such page) and slot. The position is counted from the sequence's whole length: cut to what the table
// holds, the tokens past it would take the slots, and the angles, of the newest that fit.
struct PagedPlace {
    int pos, page, slot;
};
FV_DEV PagedPlace paged_place(const PagedBatch& b, const PagedPool& pool, int t) {
    const int s = paged_seq_of(b, t);
    const PagedSeq q = paged_seq(b, s);
    const int pos = q.pos_of(max(b.lens[s], 0)) + (t - q.start);
    if (t < q.start || t >= q.start + q.count || pos < 0) return {-1, -1, 0};
    const int page = pos < b.max_len ? b.table[(size_t)s * b.table_stride + (pos >> pool.lg)] : -1;   // (max_len: the table's slots)
    return {pos, (unsigned)page < (unsigned)pool.pages ? page : -1, pos & ((1 << pool.lg) - 1)};
}

// Eight values as they stand in memory, and as f32.
template <bool IN16>
struct Eight {
    u32x4 w[IN16 ? 1 : 2];
    FV_DEV void load(const void* x, size_t at) {
        const u32x4* p = reinterpret_cast<const u32x4*>((const uint8_t*)x + at * (IN16 ? 2 : 4));
        w[0] = p[0];
        if constexpr (!IN16) w[1] = p[1];
    }
    FV_DEV void get(float (&v)[8]) const {
        if constexpr (IN16) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = __builtin_bit_cast(float, w[0][i] << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, w[0][i] & 0xffff0000u);
            }
        } else {
            // (not [i / 4][i % 4]: in one loop of eight the compiler took element 0 for 2 and 1 for 3)
            const f32x4 lo = __builtin_bit_cast(f32x4, w[0]), hi = __builtin_bit_cast(f32x4, w[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = lo[i], v[4 + i] = hi[i];
        }
    }
};
FV_DEV u32x4 to_bf16x8(const float (&r)[8]) {
    f32x8 f;
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = r[i];
    return __builtin_bit_cast(u32x4, __builtin_convertvector(f, bf16x8));
}

// The piece of eight channels that piece c of a head is turned with: its own, or (halves) that half a head away.
template <int D, bool HALVES>
FV_DEV int partner(int c) { return HALVES ? c ^ (D / 16) : c; }
// Piece `v` (the c-th) of a head and its partner `w`, turned by row `row` of the tables, f32 with unfused products (the rounding of
// the plain formula, so that the value to be stored is the same number whoever computes it).
template <bool IN16, int D, bool HALVES>
FV_DEV void turn8(const Eight<IN16>& own, const Eight<IN16>& other, int c, const float* cos_t, const float* sin_t, int row, float (&r)[8]) {
#pragma clang fp contract(off)
    const bool upper = HALVES && c >= D / 16;
    const size_t slot = (size_t)row * D + 8 * (upper ? c - D / 16 : c);
    Eight<false> ct, st;
    ct.load(cos_t, slot);
    st.load(sin_t, slot);
    float v[8], w[8], cs[8], sn[8];
    own.get(v);
    ct.get(cs);
    st.get(sn);
    if constexpr (HALVES) {   // pairs (i, i + D / 2), the angle in slot i
        other.get(w);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float x1 = upper ? w[i] : v[i], x2 = upper ? v[i] : w[i];
            r[i] = upper ? x1 * sn[i] + x2 * cs[i] : x1 * cs[i] - x2 * sn[i];
        }
    } else {                  // pairs (2 i, 2 i + 1), the angle in slot 2 i
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            r[i] = v[i] * cs[i] - v[i + 1] * sn[i];
            r[i + 1] = v[i] * sn[i] + v[i + 1] * cs[i];
        }
    }
}

// Eight values of a block of 32, which four neighbouring lanes hold, as 4-bit codes of the block's scale: 2^e, the smallest
// power of two that takes no value of the block past the largest code, 6 (so no code is off by more than half a step of its
// binade, where a scale from the exponent of the largest value alone would cut the values above 6 off). A block with a value
// that is not finite has the scale "not a number".
FV_DEV unsigned to_fp4x8(const float (&r)[8], unsigned& scale_byte) {
    float a = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        a = __builtin_fmaxf(a, __builtin_fabsf(r[i]));
        bad |= !(__builtin_fabsf(r[i]) <= 3.4028234663852886e38f);
    }
    unsigned u = bad ? 0x7f800000u : __builtin_bit_cast(unsigned, a);
    u = max(u, (unsigned)__shfl_xor((int)u, 1, 64));   // (bits of values without sign are in the values' order)
    u = max(u, (unsigned)__shfl_xor((int)u, 2, 64));
    // a = m 2^E, 1 <= m < 2: 6 2^(E - 2) = 1.5 2^E holds it where m <= 1.5, else twice that does
    const int e = (int)(u >> 23) - 2 + ((u & 0x7fffffu) > 0x400000u ? 1 : 0);
    scale_byte = u >= 0x7f800000u ? 255u : (unsigned)max(e, 1);
    const float scale = e8m0_scale(scale_byte);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[0], r[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[2], r[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[4], r[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[6], r[7], scale, 3);
    return w;
}

// Block (x, y): pieces [256 y, 256 y + 256) of token x: the query heads' first (if any), then the key heads', then the value
// heads'. 56637 tokens of 32 / 8 heads in 24 prompts, their tables and queries: 1.42 GB in 265 us, 5.4 TB/s (a large copy: 4.9; 299 with
// the values loaded behind the look-ups); 9360 of 12 heads from f32 to 4 bits: 0.14 GB in 28 us, 5.0 TB/s. 32 single tokens: 3.1 us.
template <bool IN16, int D, bool FOUR, bool HALVES>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendParams p) {
    constexpr int kPer = D / 8;
    const int piece = blockIdx.y * 256 + threadIdx.x;
    const int head = piece / kPer, c = piece % kPer, nq = p.q ? p.heads : 0, kvh = p.pool.kv_heads;
    if (head >= nq + 2 * kvh) return;
    const int t = blockIdx.x;
    const bool is_q = head < nq, turn = p.cos_t != nullptr && head < nq + kvh;
    // the values first, which wait for nothing; where they go takes four or more loads in a row
    const void* x = is_q ? p.q : head < nq + kvh ? p.k : p.v;
    const size_t from = (size_t)t * (is_q ? p.q_stride : head < nq + kvh ? p.k_stride : p.v_stride) + (is_q ? head : head < nq + kvh ? head - nq : head - nq - kvh) * D;
    Eight<IN16> own, other;
    own.load(x, from + 8 * c);
    if (HALVES && turn) other.load(x, from + 8 * partner<D, HALVES>(c));
    if (t < p.b.q_start[0] || t >= p.b.q_start[p.b.seqs]) return;   // of no sequence
    const PagedPlace at = paged_place(p.b, p.pool, t);
    const int row = p.rope_at ? p.rope_at[t] : at.pos;
    const bool ok = at.pos >= 0 && (!p.cos_t || (unsigned)row < (unsigned)p.rope_rows);
    float r[8];
    if (ok && turn) turn8<IN16, D, HALVES>(own, other, c, p.cos_t, p.sin_t, row, r);
    else own.get(r);
    if (is_q) {   // (one that lies nowhere is zeros)
        *reinterpret_cast<u32x4*>(p.q_out + ((size_t)t * p.heads + head) * D + 8 * c) = ok ? to_bf16x8(r) : u32x4{0u, 0u, 0u, 0u};
        return;
    }
    if (!ok || at.page < 0) return;
    const bool is_v = head >= nq + kvh;
    const size_t at_row = (((size_t)at.page * kvh + (head - nq - (is_v ? kvh : 0))) << p.pool.lg) + at.slot;
    uint8_t* base = (uint8_t*)(is_v ? p.pool.v : p.pool.k);
    if constexpr (FOUR) {
        unsigned scale;
        const unsigned w = to_fp4x8(r, scale);
        *reinterpret_cast<unsigned*>(base + at_row * (D / 2) + 4 * c) = w;
        if (c % 4 == 0) (is_v ? p.pool.vs : p.pool.ks)[at_row * (D / 32) + c / 4] = (uint8_t)scale;
    } else {
        *reinterpret_cast<u32x4*>(base + at_row * (2 * D) + 16 * c) = to_bf16x8(r);
    }
}

// The same walk the other way: k_out, v_out [tokens, kv_heads, d], f32 or bf16 (both exact); rows that lie nowhere are zeros. 9360
// tokens of 12 heads from 4 bits to bf16: 73 MB in 16.7 us, 4.4 TB/s.
template <bool OUT16, int D, bool FOUR>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedPool pool, const PagedBatch b, void* __restrict__ k_out, void* __restrict__ v_out) {
    constexpr int kPer = D / 8;
    const int piece = blockIdx.y * 256 + threadIdx.x, t = blockIdx.x;
    const int head = piece / kPer, c = piece % kPer, kvh = pool.kv_heads;
    if (head >= 2 * kvh) return;
    if (t < b.q_start[0] || t >= b.q_start[b.seqs]) return;   // of no sequence: left as it was
    const PagedPlace at = paged_place(b, pool, t);
    const bool is_v = head >= kvh;
    const int h = is_v ? head - kvh : head;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (at.page >= 0) {
        const size_t row = (((size_t)at.page * kvh + h) << pool.lg) + at.slot;
        const uint8_t* base = (const uint8_t*)(is_v ? pool.v : pool.k);
        if constexpr (FOUR) {
            const float scale = e8m0_scale((is_v ? pool.vs : pool.ks)[row * (D / 32) + c / 4]);
            w = fp4_eight(*reinterpret_cast<const unsigned*>(base + row * (D / 2) + 4 * c), scale);
        } else {
            w = *reinterpret_cast<const u32x4*>(base + row * (2 * D) + 16 * c);
        }
    }
    const size_t to = ((size_t)t * kvh + h) * D + 8 * c;
    void* out = is_v ? v_out : k_out;
    if constexpr (OUT16) {
        *reinterpret_cast<u32x4*>((uint16_t*)out + to) = w;
    } else {
        f32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x0 = __builtin_bit_cast(float, w[i] << 16), x1 = __builtin_bit_cast(float, w[i] & 0xffff0000u);
            if (i < 2) lo[2 * i] = x0, lo[2 * i + 1] = x1;
            else hi[2 * i - 4] = x0, hi[2 * i - 3] = x1;
        }
        *reinterpret_cast<f32x4*>((float*)out + to) = lo;
        *reinterpret_cast<f32x4*>((float*)out + to + 4) = hi;
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace fv

// The pool and the batch of a call, checked: FV_OK, or what the entry returns. `max_len`: a bound of the lengths, or null: what
// the table's columns hold.
int fv_paged_args(const char* who, const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, size_t pages,
                  size_t page_tokens, size_t kv_heads, size_t d, const int32_t* q_start, const int32_t* lens, const int32_t* table,
                  size_t table_stride, size_t table_pages, size_t seqs, size_t tokens, const size_t* max_len, fv::PagedPool* pool, fv::PagedBatch* b) {
    auto say = [who](const char* why, bool decline) {
        char buf[200];
        snprintf(buf, sizeof buf, "%s: %s", who, why);
        return decline ? fv_decline(buf) : fv_invalid(buf);
    };
    if (!k_pages || !v_pages || !q_start || !lens || !table) return say("null operand", false);
    if ((k_scales == nullptr) != (v_scales == nullptr)) return say("scales of keys and values go together (4 bits) or are both null (bf16)", false);
    if (d != 64 && d != 128) return say("head dim must be 64 or 128", true);
    if (page_tokens < 16 || (page_tokens & (page_tokens - 1)) != 0 || page_tokens > 65536)
        return say("page_tokens must be a power of two of 16 to 65536", true);
    if (kv_heads == 0 || pages == 0) return say("an empty pool", false);
    if (kv_heads > 65535 || pages > (size_t)INT_MAX) return say("pool too large", true);
    // (row numbers are 32 bits: as many rows of K and V are more than the card holds)
    if (pages > 0xffffffffull / kv_heads / page_tokens) return say("pool too large", true);
    if (!fv::aligned16(k_pages) || !fv::aligned16(v_pages) || !fv::aligned16(k_scales) || !fv::aligned16(v_scales))
        return say("pages and scales must be 16-byte aligned", false);
    if (table_pages > table_stride) return say("table rows shorter than their pages", false);
    if (table_pages > (size_t)INT_MAX / page_tokens) return say("table too wide", true);
    if (seqs > kMostSeqs || tokens > kMostRows) return say("too many sequences or rows for one launch", true);
    if (max_len && *max_len > table_pages * page_tokens) return say("lengths past the table's pages", false);
    int lg = 0;
    while (((size_t)1 << lg) < page_tokens) lg++;
    *pool = fv::PagedPool{const_cast<void*>(k_pages), const_cast<void*>(v_pages), (uint8_t*)const_cast<void*>(k_scales),
                          (uint8_t*)const_cast<void*>(v_scales), (int)pages, lg, (int)kv_heads};
    *b = fv::PagedBatch{q_start, lens, table, (long)table_stride, (int)seqs, (int)tokens,
                        (int)(max_len ? *max_len : table_pages * page_tokens)};
    return FV_OK;
}

extern "C" {

int fv_paged_append(const void* k, size_t k_stride, const void* v, size_t v_stride, const void* q, size_t q_stride, uint16_t* q_out,
                    int in_is_bf16, size_t heads, const float* cos_t, const float* sin_t, size_t rope_rows, const int32_t* rope_at,
                    int halves, void* k_pages, void* v_pages, void* k_scales, void* v_scales, size_t pages, size_t page_tokens,
                    size_t kv_heads, size_t d, const int32_t* q_start, const int32_t* lens, const int32_t* table, size_t table_stride,
                    size_t table_pages, size_t seqs, size_t tokens, void* stream) {
    if (seqs == 0 || tokens == 0) return FV_OK;   // (empty arrays may have no address)
    fv::AppendParams p;
    const int rc = fv_paged_args("paged append", k_pages, v_pages, k_scales, v_scales, pages, page_tokens, kv_heads, d, q_start, lens, table,
                                 table_stride, table_pages, seqs, tokens, nullptr, &p.pool, &p.b);
    if (rc != FV_OK) return rc;
    if (!k || !v) return fv_invalid("paged append: null operand");
    if ((q == nullptr) != (q_out == nullptr)) return fv_invalid("paged append: queries without a place for the rotated ones, or the reverse");
    if ((cos_t == nullptr) != (sin_t == nullptr)) return fv_invalid("paged append: one rope table without the other");
    if (q && heads == 0) return fv_invalid("paged append: queries without heads");
    const size_t most = (size_t)INT_MAX / 4;
    if (heads > 65535) return fv_decline("paged append: too many heads");
    if (k_stride < kv_heads * d || v_stride < kv_heads * d || (q && q_stride < heads * d))
        return fv_invalid("paged append: tokens overlap (a stride below heads * d)");
    if (k_stride % 8 != 0 || v_stride % 8 != 0 || (q && q_stride % 8 != 0) || k_stride > most || v_stride > most || (q && q_stride > most))
        return fv_decline("paged append: strides must be multiples of 8 elements");
    if (!fv::aligned16(k) || !fv::aligned16(v) || !fv::aligned16(q) || !fv::aligned16(q_out) || !fv::aligned16(cos_t) || !fv::aligned16(sin_t))
        return fv_invalid("paged append: operands must be 16-byte aligned");
    if (rope_rows > (size_t)INT_MAX) return fv_decline("paged append: rope tables too long");
    p.k = k, p.v = v, p.q = q, p.q_out = q_out;
    p.k_stride = (long)k_stride, p.v_stride = (long)v_stride, p.q_stride = (long)q_stride;
    p.cos_t = cos_t, p.sin_t = sin_t, p.rope_at = rope_at, p.rope_rows = (int)rope_rows, p.heads = (int)heads;
    const size_t pieces = ((q ? heads : 0) + 2 * kv_heads) * (d / 8);
    const dim3 grid((unsigned)tokens, (unsigned)((pieces + 255) / 256));
    if ((size_t)grid.x * grid.y >= (size_t)1 << 24) return fv_decline("paged append: too large for one launch");
    const bool four = k_scales != nullptr;
    hipStream_t st = (hipStream_t)stream;
    fv::paged_pick(in_is_bf16 != 0, [&](auto i16) {
        fv::paged_pick(d == 128, [&](auto d128) {
            fv::paged_pick(four, [&](auto f) {
                fv::paged_pick(halves != 0, [&](auto h) {
                    hipLaunchKernelGGL((fv::paged_append_kernel<i16(), d128() ? 128 : 64, f(), h()>), grid, dim3(256), 0, st, p);
                });
            });
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "paged_append");
}

int fv_paged_read(void* k_out, void* v_out, int out_is_bf16, const void* k_pages, const void* v_pages, const void* k_scales,
                  const void* v_scales, size_t pages, size_t page_tokens, size_t kv_heads, size_t d, const int32_t* q_start,
                  const int32_t* lens, const int32_t* table, size_t table_stride, size_t table_pages, size_t seqs, size_t tokens,
                  void* stream) {
    if (seqs == 0 || tokens == 0) return FV_OK;
    fv::PagedPool pool;
    fv::PagedBatch b;
    const int rc = fv_paged_args("paged read", k_pages, v_pages, k_scales, v_scales, pages, page_tokens, kv_heads, d, q_start, lens, table,
                                 table_stride, table_pages, seqs, tokens, nullptr, &pool, &b);
    if (rc != FV_OK) return rc;
    if (!k_out || !v_out) return fv_invalid("paged read: null operand");
    if (!fv::aligned16(k_out) || !fv::aligned16(v_out)) return fv_invalid("paged read: operands must be 16-byte aligned");
    const dim3 grid((unsigned)tokens, (unsigned)((2 * kv_heads * (d / 8) + 255) / 256));
    if ((size_t)grid.x * grid.y >= (size_t)1 << 24) return fv_decline("paged read: too large for one launch");
    const bool four = k_scales != nullptr;
    hipStream_t st = (hipStream_t)stream;
    fv::paged_pick(out_is_bf16 != 0, [&](auto o16) {
        fv::paged_pick(d == 128, [&](auto d128) {
            fv::paged_pick(four, [&](auto f) {
                hipLaunchKernelGGL((fv::paged_read_kernel<o16(), d128() ? 128 : 64, f()>), grid, dim3(256), 0, st, pool, b, k_out, v_out);
            });
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FV_OK : fv_fail_hip(e, "paged_read");
}

}  // extern "C"
