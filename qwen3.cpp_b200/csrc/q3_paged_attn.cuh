// What the kernels of q3_paged_attn / q3_prefix_attn share: arguments, the partition of the work over
// a sequence's own pages, and the layout of the workspace.
#pragma once

#include "q3_paged.cuh"

namespace q3 {

struct PagedArgs {
    void* out;
    const void* q;
    const void* k;
    const void* v;
    const uint8_t* exps;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* table;
    const int32_t* prefix_table;
    long long q_stride, out_stride;
    int n_pages, n_kv, group, n_q, n_seqs, max_q, table_stride, prefix_len;
    unsigned group_magic;  // ceil(2^32 / group), 0 for a group of one: see token_of
    int f16;         // q and out are fp16 (else bf16)
    // Workspace. Partial results are in fp32: o = sum p v and (m, l) = (max of the scores in units of
    // log2, sum p), p = 2^(score - m + kShift).
    float* own_o;           // [blocks][2][8 * tiles][head_dim]
    float2* own_ml;         // [blocks][2][8 * tiles]
    float* whole_o;         // [n_kv][prefix_rows][head_dim]: with a prefix, own parts that were not cut
    float2* whole_ml;       // [n_kv][prefix_rows]
    float* prefix_o;        // [splits][n_kv][prefix_rows][head_dim]
    float2* prefix_ml;      // [splits][n_kv][prefix_rows]
    int prefix_splits, prefix_rows;
    int inline_pages;       // of the prefix, where the strips read them themselves (prefix_splits is 0 then)
};

constexpr float kShift = 8.0f;     // the weights' largest is about 2^8: fp16 then reaches to 2^-32 of it
constexpr int kMaxBlocks = 640;    // of the line: at least 4 a multiprocessor
constexpr int kSetup = 16;         // what a strip costs beside its pages, in pages (4: 64 sequences 60 us, 8: 56, 16: 54, 24: 55)
constexpr int kMinUnits = 12;      // a block's smallest share

// Rows of sequence b and its own tokens, whatever the arrays hold.
struct SeqShape {
    int row0, rows, len;
};
__device__ __forceinline__ SeqShape seq_shape(const PagedArgs& a, int b) {
    SeqShape s;
    s.row0 = min(max(a.q_start[b], 0), a.n_q);
    s.rows = min(min(a.q_start[b + 1], a.n_q) - s.row0, a.max_q);
    s.rows = max(s.rows, 0);
    s.len = static_cast<int>(min(static_cast<long long>(max(a.kv_len[b], 0)),
                                 static_cast<long long>(a.table_stride) * kPageTokens));
    return s;
}

// The query token of row r of a KV head, r / group (its head of the group is r % group): exact for rows
// below 2^26, as magic * group is less than 2^32 + 64.
__device__ __forceinline__ int token_of(const PagedArgs& a, int r) {
    return a.group_magic ? static_cast<int>(__umulhi(static_cast<unsigned>(r), a.group_magic)) : r;
}

__device__ __forceinline__ int seq_pages(const SeqShape& s) {
    return static_cast<int>((static_cast<long long>(s.len) + kPageTokens - 1) / kPageTokens);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^e for any int e (0 below the normal range, infinity above).
__device__ __forceinline__ float pow2(int e) {
    return e < -126 ? 0.0f : e > 127 ? INFINITY : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ uint32_t pack2_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two weights as hi + lo in bf16, for a bf16 pool. hi is the weight cut off, and lo the rest with 2^-23 of the
// weight on top, rounded (2^-16 of the weight): both are positive where the weight is, so that an infinite value
// times them is that infinity. (A rounded hi leaves a lo of zero or less for half of the weights, and NaN.)
__device__ __forceinline__ uint32_t weights_hi(float x, float y) {
    return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632u);
}
__device__ __forceinline__ uint32_t weights_lo(float x, float y, uint32_t hi) {
    constexpr float kOnTop = 1.00000011920928955078125f;  // 1 + 2^-23
    return pack2_bf16(fmaf(x, kOnTop, -bf16_lo(hi)), fmaf(y, kOnTop, -bf16_hi(hi)));
}
// Two results in the caller's type, to nearest even; an fp16 result past the range becomes infinity.
__device__ __forceinline__ uint32_t pack2_out(float lo, float hi, int f16) {
    if (!f16) return pack2_bf16(lo, hi);
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

void launch_prefix_attention(const PagedArgs& a, int head_dim, bool e4m3, cudaStream_t s);
// Parts that the prefix kernel leaves for each row, from the sizes alone.
int prefix_splits(int n_kv, int rows, int prefix_len);
// The most parts, of all rows together, that a batch of so many rows or fewer leaves over a prefix of this
// length or a shorter one.
size_t prefix_part_rows(int n_kv, int rows, int prefix_len);

}  // namespace q3
