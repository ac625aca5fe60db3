// q3_paged_attn / q3_prefix_attn: attention of a ragged batch's newest rows over a paged KV pool,
// with or without a prefix that every sequence shares.
#include <climits>

#include "q3_paged.cuh"

namespace q3 {

namespace {

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
    int n_pages, n_kv, group, n_q, n_seqs, max_q, table_stride, prefix_len, f16, e4m3;
};

__device__ __forceinline__ float value16(const void* p, size_t i, int f16) {
    const uint16_t u = static_cast<const uint16_t*>(p)[i];
    return f16 ? __half2float(__ushort_as_half(u)) : bf16_to_f32(u);
}

// One warp per (row, query head), a lane per D / 32 values of the head.
template <int D>
__global__ void __launch_bounds__(128) attn_rows_kernel(const PagedArgs a) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, heads = a.n_kv * a.group;
    const int head = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int b = blockIdx.x / a.max_q, i = blockIdx.x % a.max_q;
    if (head >= heads) return;
    const int r0 = max(a.q_start[b], 0), r1 = min(a.q_start[b + 1], a.n_q);
    const int rows = min(r1 - r0, a.max_q);
    if (i >= rows) return;
    const int kvh = head / a.group;
    const int len = static_cast<int>(
        min(static_cast<long long>(max(a.kv_len[b], 0)), static_cast<long long>(a.table_stride) * kPageTokens));
    const int seen = max(0, len - rows + i + 1);
    float q[V], o[V] = {};
#pragma unroll
    for (int d = 0; d < V; ++d) {
        q[d] = value16(a.q, (r0 + i) * a.q_stride + head * D + lane * V + d, a.f16) *
               (1.4426950408889634f / sqrtf(static_cast<float>(D)));
    }
    float m = -INFINITY, l = 0.0f;
    for (int part = 0; part < 2; ++part) {
        const int32_t* table = part ? a.table + static_cast<size_t>(b) * a.table_stride : a.prefix_table;
        const int keys = part ? seen : a.prefix_len;
        for (int j = 0; j < keys; ++j) {
            const int page = table[j / kPageTokens];
            if (page < 0 || page >= a.n_pages) continue;
            const size_t row = (static_cast<size_t>(page) * a.n_kv + kvh) * kPageTokens + j % kPageTokens;
            float kx[V], vx[V];
#pragma unroll
            for (int d = 0; d < V; ++d) {
                const size_t at = row * D + lane * V + d;
                if (a.e4m3) {
                    kx[d] = f16_lo(e4m3x2_to_f16x2(static_cast<const uint8_t*>(a.k)[at])) *
                            exp_of_byte(a.exps[row * 2]);
                    vx[d] = f16_lo(e4m3x2_to_f16x2(static_cast<const uint8_t*>(a.v)[at])) *
                            exp_of_byte(a.exps[row * 2 + 1]);
                } else {
                    kx[d] = bf16_to_f32(static_cast<const uint16_t*>(a.k)[at]);
                    vx[d] = bf16_to_f32(static_cast<const uint16_t*>(a.v)[at]);
                }
            }
            float s = 0.0f;
#pragma unroll
            for (int d = 0; d < V; ++d) s = fmaf(q[d], kx[d], s);
            s = warp_sum(s);
            const float m_new = fmaxf(m, s);
            const float f = m_new == -INFINITY ? 1.0f : exp2f(m - m_new);
            const float p = m_new == -INFINITY ? 0.0f : exp2f(s - m_new);
            l = l * f + p;
#pragma unroll
            for (int d = 0; d < V; ++d) o[d] = fmaf(p, vx[d], o[d] * f);
            m = m_new;
        }
    }
#pragma unroll
    for (int d = 0; d < V; ++d) {
        const float y = l == 0.0f ? 0.0f : o[d] / l;  // a row that sees nothing is zeros
        static_cast<uint16_t*>(a.out)[(r0 + i) * a.out_stride + head * D + lane * V + d] =
            a.f16 ? __half_as_ushort(__float2half_rn(y)) : f32_to_bf16(y);
    }
}

constexpr int kMaxGroup = 64, kMaxRows = 128;

bool sizes_ok(const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs, int max_q, int prefix_len) {
    return n_heads > 0 && n_heads % pool->n_kv_heads == 0 && n_heads / pool->n_kv_heads <= kMaxGroup &&
           n_q >= 0 && n_seqs >= 0 && max_q > 0 &&
           static_cast<long long>(max_q) * (n_heads / pool->n_kv_heads) <= kMaxRows && prefix_len >= 0;
}

void paged_attention(void* out, void* workspace, const void* q, int type, int64_t q_stride,
                     int64_t out_stride, const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs,
                     int max_q, const int32_t* q_start, const int32_t* kv_len, const int32_t* table,
                     int table_stride, const int32_t* prefix_table, int prefix_len, void* stream) {
    check_pool(pool);
    if (type != Q3_TYPE_BF16 && !(type == Q3_TYPE_F16 && pool->type == Q3_TYPE_E4M3)) {
        throw std::invalid_argument("paged attention: type must be BF16, or F16 with an e4m3 pool");
    }
    if (!sizes_ok(pool, n_heads, n_q, n_seqs, max_q, prefix_len) || table_stride < 0) {
        throw std::invalid_argument("paged attention: size out of range");
    }
    if (n_q == 0 || n_seqs == 0) return;
    if (!out || !workspace || !q || !q_start || !kv_len || (table_stride > 0 && !table) ||
        (prefix_len > 0 && !prefix_table)) {
        throw std::invalid_argument("paged attention: null pointer");
    }
    const int64_t width = static_cast<int64_t>(n_heads) * pool->head_dim;
    if (q_stride < width || out_stride < width || q_stride % 8 != 0 || out_stride % 8 != 0) {
        throw std::invalid_argument(
            "paged attention: strides must cover n_heads * head_dim and be multiples of 8");
    }
    if (!aligned(out, 16) || !aligned(q, 16) || !aligned(workspace, 16) || !aligned(q_start, 4) ||
        !aligned(kv_len, 4) || !aligned(table, 4) || !aligned(prefix_table, 4)) {
        throw std::invalid_argument("paged attention: misaligned pointer");
    }
    const OnDevice on({out, workspace, q, pool->k, pool->v, pool->exps, q_start, kv_len,
                       table_stride ? table : nullptr, prefix_len ? prefix_table : nullptr});
    PagedArgs a{};
    a.out = out;
    a.q = q;
    a.k = pool->k;
    a.v = pool->v;
    a.exps = pool->exps;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.table = table;
    a.prefix_table = prefix_table;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n_pages = static_cast<int>(pool->n_pages);
    a.n_kv = pool->n_kv_heads;
    a.group = n_heads / pool->n_kv_heads;
    a.n_q = n_q;
    a.n_seqs = n_seqs;
    a.max_q = max_q;
    a.table_stride = table_stride;
    a.prefix_len = prefix_len;
    a.f16 = type == Q3_TYPE_F16;
    a.e4m3 = pool->type == Q3_TYPE_E4M3;
    const dim3 grid(n_seqs * max_q, (n_heads + 3) / 4);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    launch_dep(false, pool->head_dim == 64 ? attn_rows_kernel<64> : attn_rows_kernel<128>, grid,
               dim3(128), 0, s, a);
}

}  // namespace

}  // namespace q3

extern "C" {

size_t q3_paged_attn_workspace_size(const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs,
                                    int max_q, int prefix_len) {
    if (!pool || pool->n_kv_heads <= 0 || (pool->head_dim != 64 && pool->head_dim != 128) ||
        !q3::sizes_ok(pool, n_heads, n_q, n_seqs, max_q, prefix_len)) {
        return 0;
    }
    return 256;
}

q3_status q3_paged_attn(void* out, void* workspace, const void* q, int type, int64_t q_stride,
                        int64_t out_stride, const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs,
                        int max_q, const int32_t* q_start, const int32_t* kv_len,
                        const int32_t* table, int table_stride, void* stream) {
    return q3::guard([&] {
        q3::paged_attention(out, workspace, q, type, q_stride, out_stride, pool, n_heads, n_q, n_seqs,
                            max_q, q_start, kv_len, table, table_stride, nullptr, 0, stream);
    });
}

q3_status q3_prefix_attn(void* out, void* workspace, const void* q, int type, int64_t q_stride,
                         int64_t out_stride, const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs,
                         int max_q, const int32_t* q_start, const int32_t* kv_len,
                         const int32_t* table, int table_stride, const int32_t* prefix_table,
                         int prefix_len, void* stream) {
    return q3::guard([&] {
        q3::paged_attention(out, workspace, q, type, q_stride, out_stride, pool, n_heads, n_q, n_seqs,
                            max_q, q_start, kv_len, table, table_stride, prefix_table, prefix_len,
                            stream);
    });
}

}  // extern "C"
