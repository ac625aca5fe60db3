// q3_kv_write / q3_kv_read: rows of a paged KV pool quantised as they are written, and read back.
//
// An e4m3 row x[0..head_dim) is stored as codes c and one byte b with x ~ c * 2^(b - 127). b is the
// smallest byte with amax <= 448 * 2^(b - 127) (448 is the largest e4m3 value), read off amax's
// exponent and fraction: amax = f * 2^E, 1 <= f < 2, needs b - 127 = E - 8 for f <= 1.75 (448 = 1.75 *
// 2^8) and E - 7 above. A power of two makes the scaling exact, so the only rounding is the one to
// e4m3 (relative 2^-4) and the codes do not depend on how a product would round. One byte a row costs
// 1 / head_dim of the codes.
//
// Both directions are bound by HBM: 2 * H * (size * D + D + 1) bytes a token (4096 tokens of 8 heads of
// 128 written from bf16: 5.4 us, 25 MB). A group of D / V lanes
// takes HEADS heads of a token: V consecutive values a lane of each K row and V row, amax by shuffles
// inside the group, and a row's two bytes stored as one 16-bit word.
#include "q3_paged.cuh"

namespace q3 {

namespace {

struct RowsArgs {
    void* pool_k;
    void* pool_v;
    uint8_t* exps;
    void* k;  // the caller's rows: written from (kv_write) or to (kv_read)
    void* v;
    const int32_t* slots;
    long long k_stride, v_stride, n_slots;
    int n, n_kv;
};

template <int TYPE>
struct Elem;
template <>
struct Elem<Q3_TYPE_F32> {
    using T = float;
    static __device__ __forceinline__ float get(T x) { return x; }
};
template <>
struct Elem<Q3_TYPE_BF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float get(T x) { return bf16_to_f32(x); }
};
template <>
struct Elem<Q3_TYPE_F16> {
    using T = uint16_t;
    static __device__ __forceinline__ float get(T x) { return __half2float(__ushort_as_half(x)); }
};

// Two values in 16 bits each, to nearest even.
template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (TYPE == Q3_TYPE_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// V consecutive elements; VEC: their address is a multiple of 16 bytes (or of their size together).
template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_run(const T* p, T (&x)[V]) {
    if constexpr (VEC) {
        constexpr int W = V * sizeof(T) >= 16 ? 16 : V * sizeof(T);
        static_assert(W == 16 || W == 8, "run width");
#pragma unroll
        for (int i = 0; i < V; i += W / sizeof(T)) {
            if constexpr (W == 16) *reinterpret_cast<uint4*>(x + i) = *reinterpret_cast<const uint4*>(p + i);
            else *reinterpret_cast<uint2*>(x + i) = *reinterpret_cast<const uint2*>(p + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p[i];
    }
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_run(T* p, const T (&x)[V]) {
    if constexpr (VEC) {
        constexpr int W = V * sizeof(T) >= 16 ? 16 : V * sizeof(T);
        static_assert(W == 16 || W == 8, "run width");
#pragma unroll
        for (int i = 0; i < V; i += W / sizeof(T)) {
            if constexpr (W == 16) *reinterpret_cast<uint4*>(p + i) = *reinterpret_cast<const uint4*>(x + i);
            else *reinterpret_cast<uint2*>(p + i) = *reinterpret_cast<const uint2*>(x + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = x[i];
    }
}

constexpr int kThreads = 128;
constexpr long long kManyLanes = 1 << 18;

// HEADS: heads of one token that a group of lanes takes, with one slot look-up and 2 * HEADS
// independent loads a lane. 4 where the rows fill the GPU's lanes several times (8 heads of 128, 32768
// tokens read as bf16: 35.9 us, 87% of the copy rate, against 42.1 with 1), 1 below that (1 token written: 1.5 us against 2.4).

// Element offset of (slot, head)'s row in the pool.
template <int D>
__device__ __forceinline__ size_t pool_row(long long slot, int head, int n_kv) {
    return ((static_cast<size_t>(slot / kPageTokens) * n_kv + head) * kPageTokens +
            slot % kPageTokens) * D;
}

// This lane's token, first head and first value of the head; false past the last token.
template <int D, int V, int HEADS>
__device__ __forceinline__ bool my_place(const RowsArgs& a, int& token, int& head, int& d) {
    constexpr unsigned LANES = D / V;
    const unsigned at = blockIdx.x * kThreads + threadIdx.x, group = at / LANES;
    const unsigned per_token = (a.n_kv + HEADS - 1) / HEADS;
    token = static_cast<int>(group / per_token);
    head = static_cast<int>(group % per_token) * HEADS;
    d = static_cast<int>(at % LANES) * V;
    return token < a.n;
}

template <int TYPE, int D, bool E4M3, bool VEC, int HEADS>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const RowsArgs a) {
    using E = Elem<TYPE>;
    using T = typename E::T;
    constexpr int V = 8, LANES = D / V;
    int token, head0, d;
    // Whole groups share their place, so a group is in or out of range together; its lanes stay for the
    // shuffles of the warp's other groups.
    const long long slot = my_place<D, V, HEADS>(a, token, head0, d) ? a.slots[token] : -1;
    const bool live = slot >= 0 && slot < a.n_slots;
    const size_t to0 = live ? pool_row<D>(slot, head0, a.n_kv) : 0;
    alignas(16) T raw[HEADS][2][V];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (live && head0 + h < a.n_kv) {
            const size_t from = static_cast<size_t>(head0 + h) * D + d;
            load_run<T, V, VEC>(static_cast<const T*>(a.k) + token * a.k_stride + from, raw[h][0]);
            load_run<T, V, VEC>(static_cast<const T*>(a.v) + token * a.v_stride + from, raw[h][1]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) raw[h][0][i] = raw[h][1][i] = T{};
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        const bool here = live && head0 + h < a.n_kv;
        const size_t to = to0 + static_cast<size_t>(h) * kPageTokens * D;
        uint32_t bytes = 0;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float x[V];
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = E::get(raw[h][w][i]);
            if constexpr (E4M3) {
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float m = fabsf(x[i]);
                    if (m < INFINITY) big = fmaxf(big, m);  // false for NaN
                }
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) {
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                }
                const uint32_t bits = __float_as_uint(big);
                const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
                const uint32_t byte = static_cast<uint32_t>(max(e, 0));
                const float scale = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
                uint32_t c[V / 4];
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(
                        make_float2(x[i] * scale, x[i + 1] * scale), __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
                        make_float2(x[i + 2] * scale, x[i + 3] * scale), __NV_SATFINITE, __NV_E4M3);
                    c[i / 4] = lo | hi << 16;
                }
                bytes |= byte << (8 * w);
                uint8_t* pool = static_cast<uint8_t*>(w ? a.pool_v : a.pool_k);
                if (here) *reinterpret_cast<uint2*>(pool + to + d) = make_uint2(c[0], c[1]);
            } else {
                uint32_t c[V / 2];
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    c[i / 2] = pack2<Q3_TYPE_BF16>(x[i], x[i + 1]);
                }
                uint16_t* pool = static_cast<uint16_t*>(w ? a.pool_v : a.pool_k);
                if (here) *reinterpret_cast<uint4*>(pool + to + d) = make_uint4(c[0], c[1], c[2], c[3]);
            }
        }
        if (E4M3 && here && d == 0) {
            reinterpret_cast<uint16_t*>(a.exps)[to / D] = static_cast<uint16_t>(bytes);
        }
    }
}

template <int TYPE, int D, bool E4M3, bool VEC, int HEADS>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const RowsArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int V = 16 / sizeof(T);            // one 16-byte store a lane
    constexpr int W = E4M3 ? V / 4 : V / 2;      // words that it reads for them
    int token, head0, d;
    if (!my_place<D, V, HEADS>(a, token, head0, d)) return;
    const long long slot = a.slots[token];
    const bool live = slot >= 0 && slot < a.n_slots;
    const size_t from0 = live ? pool_row<D>(slot, head0, a.n_kv) : 0;
    alignas(16) uint32_t c[HEADS][2][W];
    uint32_t bytes[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        const bool here = live && head0 + h < a.n_kv;
        const size_t from = from0 + static_cast<size_t>(h) * kPageTokens * D;
        bytes[h] = E4M3 && here ? reinterpret_cast<const uint16_t*>(a.exps)[from / D] : 0;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint8_t* p = static_cast<const uint8_t*>(w ? a.pool_v : a.pool_k) + (from + d) * (E4M3 ? 1 : 2);
#pragma unroll
            for (int i = 0; i < W; ++i) c[h][w][i] = 0;
            if (here) {
                if constexpr (W == 4) *reinterpret_cast<uint4*>(c[h][w]) = *reinterpret_cast<const uint4*>(p);
                else if constexpr (W == 2) *reinterpret_cast<uint2*>(c[h][w]) = *reinterpret_cast<const uint2*>(p);
                else c[h][w][0] = *reinterpret_cast<const uint32_t*>(p);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (head0 + h >= a.n_kv) break;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float x[V];
            if constexpr (E4M3) {
                const float f = exp_of_byte((bytes[h] >> (8 * w)) & 0xffu);
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const uint32_t lo = e4m3x2_to_f16x2(c[h][w][i / 4]), hi = e4m3x2_hi_to_f16x2(c[h][w][i / 4]);
                    x[i] = f16_lo(lo) * f;
                    x[i + 1] = f16_hi(lo) * f;
                    x[i + 2] = f16_lo(hi) * f;
                    x[i + 3] = f16_hi(hi) * f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    x[i] = bf16_lo(c[h][w][i / 2]);
                    x[i + 1] = bf16_hi(c[h][w][i / 2]);
                }
            }
            alignas(16) T y[V];
            if constexpr (TYPE == Q3_TYPE_F32) {
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = x[i];
            } else {
#pragma unroll
                for (int i = 0; i < V; i += 2) reinterpret_cast<uint32_t*>(y)[i / 2] = pack2<TYPE>(x[i], x[i + 1]);
            }
            T* to = static_cast<T*>(w ? a.v : a.k) + token * (w ? a.v_stride : a.k_stride) +
                    static_cast<size_t>(head0 + h) * D + d;
            store_run<T, V, VEC>(to, y);
        }
    }
}

template <int TYPE, int D, bool E4M3, int HEADS>
void launch_rows(bool write, bool vec, const RowsArgs& a, cudaStream_t s) {
    const int per = write ? 8 : 16 / static_cast<int>(sizeof(typename Elem<TYPE>::T));
    const long long threads = static_cast<long long>(a.n) * ((a.n_kv + HEADS - 1) / HEADS) * (D / per);
    if (threads > 0xffffff00LL) throw std::invalid_argument("KV rows: too many in one call");
    const dim3 grid(static_cast<unsigned>((threads + kThreads - 1) / kThreads));
    auto kernel = write ? (vec ? kv_write_kernel<TYPE, D, E4M3, true, HEADS> : kv_write_kernel<TYPE, D, E4M3, false, HEADS>)
                        : (vec ? kv_read_kernel<TYPE, D, E4M3, true, HEADS> : kv_read_kernel<TYPE, D, E4M3, false, HEADS>);
    launch_dep(false, kernel, grid, dim3(kThreads), 0, s, a);
}

template <int TYPE, int D, bool E4M3>
void launch_rows(bool write, bool vec, const RowsArgs& a, cudaStream_t s) {
    if (static_cast<long long>(a.n) * a.n_kv * (D / 8) >= kManyLanes) launch_rows<TYPE, D, E4M3, 4>(write, vec, a, s);
    else launch_rows<TYPE, D, E4M3, 1>(write, vec, a, s);
}

template <int TYPE>
void launch_rows(bool write, bool vec, const q3_kv_pool* pool, const RowsArgs& a, cudaStream_t s) {
    const bool e4m3 = pool->type == Q3_TYPE_E4M3;
    if (pool->head_dim == 64) {
        e4m3 ? launch_rows<TYPE, 64, true>(write, vec, a, s) : launch_rows<TYPE, 64, false>(write, vec, a, s);
    } else {
        e4m3 ? launch_rows<TYPE, 128, true>(write, vec, a, s) : launch_rows<TYPE, 128, false>(write, vec, a, s);
    }
}

void kv_rows(bool write, const q3_kv_pool* pool, void* k, void* v, int type, int64_t k_stride,
             int64_t v_stride, const int32_t* slots, int n, void* stream) {
    check_pool(pool);
    if (type != Q3_TYPE_F32 && type != Q3_TYPE_BF16 && type != Q3_TYPE_F16) {
        throw std::invalid_argument("KV rows: type must be F32, BF16 or F16");
    }
    if (n < 0) throw std::invalid_argument("KV rows: negative count");
    if (n == 0) return;
    if (!k || !v || !slots) throw std::invalid_argument("KV rows: null pointer");
    const size_t size = type == Q3_TYPE_F32 ? 4 : 2;
    const int64_t width = static_cast<int64_t>(pool->n_kv_heads) * pool->head_dim;
    if (k_stride < width || v_stride < width) {
        throw std::invalid_argument("KV rows: stride below n_kv_heads * head_dim");
    }
    if (!aligned(k, size) || !aligned(v, size) || !aligned(slots, 4)) {
        throw std::invalid_argument("KV rows: misaligned pointer");
    }
    const OnDevice on({pool->k, pool->v, pool->exps, k, v, slots});
    RowsArgs a{pool->k, pool->v, pool->exps, k, v, slots, k_stride, v_stride,
               static_cast<long long>(pool->n_pages) * kPageTokens, n, pool->n_kv_heads};
    // Rows that start on 16-byte boundaries move in 16-byte pieces, others value by value.
    const bool vec = aligned(k, 16) && aligned(v, 16) && k_stride * size % 16 == 0 &&
                     v_stride * size % 16 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == Q3_TYPE_F32) launch_rows<Q3_TYPE_F32>(write, vec, pool, a, s);
    else if (type == Q3_TYPE_BF16) launch_rows<Q3_TYPE_BF16>(write, vec, pool, a, s);
    else launch_rows<Q3_TYPE_F16>(write, vec, pool, a, s);
}

}  // namespace

}  // namespace q3

extern "C" {

q3_status q3_kv_write(const q3_kv_pool* pool, const void* k, const void* v, int type,
                      int64_t k_stride, int64_t v_stride, const int32_t* slots, int n,
                      void* stream) {
    return q3::guard([&] {
        q3::kv_rows(true, pool, const_cast<void*>(k), const_cast<void*>(v), type, k_stride, v_stride,
                    slots, n, stream);
    });
}

q3_status q3_kv_read(const q3_kv_pool* pool, void* k, void* v, int type, int64_t k_stride,
                     int64_t v_stride, const int32_t* slots, int n, void* stream) {
    return q3::guard([&] {
        q3::kv_rows(false, pool, k, v, type, k_stride, v_stride, slots, n, stream);
    });
}

}  // extern "C"
