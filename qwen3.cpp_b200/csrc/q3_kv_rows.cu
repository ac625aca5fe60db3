// q3_kv_write / q3_kv_read: rows of a paged KV pool quantised as they are written, and read back.
//
// An e4m3 row x[0..head_dim) is stored as codes c and one byte b with x ~ c * 2^(b - 127). b is the
// smallest byte with amax <= 448 * 2^(b - 127) (448 is the largest e4m3 value), read off amax's
// exponent and fraction: amax = f * 2^E, 1 <= f < 2, needs b - 127 = E - 8 for f <= 1.75 (448 = 1.75 *
// 2^8) and E - 7 above. A power of two makes the scaling exact, so the only rounding is the one to
// e4m3 (relative 2^-4) and the codes do not depend on how a product would round. One byte a row costs
// 1 / head_dim of the codes.
//
// Both directions are bound by HBM: 2 * H * (size * D + D + 1) bytes a token. A group of D / V lanes
// takes one (token, head): V consecutive values a lane of the K row and of the V row, two loads in
// flight, amax by shuffles inside the group, and the row's two bytes stored as one 16-bit word.
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
    static __device__ __forceinline__ T put(float x) { return x; }
};
template <>
struct Elem<Q3_TYPE_BF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float get(T x) { return bf16_to_f32(x); }
    static __device__ __forceinline__ T put(float x) { return f32_to_bf16(x); }
};
template <>
struct Elem<Q3_TYPE_F16> {
    using T = uint16_t;
    static __device__ __forceinline__ float get(T x) { return __half2float(__ushort_as_half(x)); }
    static __device__ __forceinline__ T put(float x) { return __half_as_ushort(__float2half_rn(x)); }
};

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

constexpr int kThreads = 256;

// Element offset of (slot, head)'s row in the pool.
template <int D>
__device__ __forceinline__ size_t pool_row(long long slot, int head, int n_kv) {
    return ((static_cast<size_t>(slot / kPageTokens) * n_kv + head) * kPageTokens +
            slot % kPageTokens) * D;
}

template <int TYPE, int D, bool E4M3, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const RowsArgs a) {
    using E = Elem<TYPE>;
    using T = typename E::T;
    constexpr int V = 8, LANES = D / V;
    const long long at = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    const long long row = at / LANES;  // (token, head)
    const int token = static_cast<int>(row / a.n_kv), head = static_cast<int>(row % a.n_kv);
    const int d = static_cast<int>(at % LANES) * V;
    // Whole groups share `token`, so a group is in or out of range together; its lanes stay for the
    // shuffles of the warp's other groups.
    const long long slot = token < a.n ? a.slots[token] : -1;
    const bool live = slot >= 0 && slot < a.n_slots;
    T raw[2][V] = {};
    if (live) {
        load_run<T, V, VEC>(static_cast<const T*>(a.k) + token * a.k_stride + head * D + d, raw[0]);
        load_run<T, V, VEC>(static_cast<const T*>(a.v) + token * a.v_stride + head * D + d, raw[1]);
    }
    const size_t to = live ? pool_row<D>(slot, head, a.n_kv) : 0;
    uint32_t bytes = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = E::get(raw[w][i]);
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
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[i] * scale, x[i + 1] * scale),
                                                             __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(
                    make_float2(x[i + 2] * scale, x[i + 3] * scale), __NV_SATFINITE, __NV_E4M3);
                c[i / 4] = lo | hi << 16;
            }
            bytes |= byte << (8 * w);
            uint8_t* pool = static_cast<uint8_t*>(w ? a.pool_v : a.pool_k);
            if (live) *reinterpret_cast<uint2*>(pool + to + d) = make_uint2(c[0], c[1]);
        } else {
            uint32_t c[V / 2];
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                c[i / 2] = f32_to_bf16(x[i]) | static_cast<uint32_t>(f32_to_bf16(x[i + 1])) << 16;
            }
            uint16_t* pool = static_cast<uint16_t*>(w ? a.pool_v : a.pool_k);
            if (live) *reinterpret_cast<uint4*>(pool + to + d) = make_uint4(c[0], c[1], c[2], c[3]);
        }
    }
    if (E4M3 && live && d == 0) {
        reinterpret_cast<uint16_t*>(a.exps)[to / D] = static_cast<uint16_t>(bytes);
    }
}

template <int TYPE, int D, bool E4M3, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const RowsArgs a) {
    using E = Elem<TYPE>;
    using T = typename E::T;
    constexpr int V = 16 / sizeof(T), LANES = D / V;  // one 16-byte store a lane
    const long long at = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    const long long row = at / LANES;
    const int token = static_cast<int>(row / a.n_kv), head = static_cast<int>(row % a.n_kv);
    const int d = static_cast<int>(at % LANES) * V;
    if (token >= a.n) return;
    const long long slot = a.slots[token];
    float x[2][V] = {};
    if (slot >= 0 && slot < a.n_slots) {
        const size_t from = pool_row<D>(slot, head, a.n_kv);
        if constexpr (E4M3) {
            const uint32_t bytes = reinterpret_cast<const uint16_t*>(a.exps)[from / D];
            uint32_t c[2][V / 4];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint8_t* p = static_cast<const uint8_t*>(w ? a.pool_v : a.pool_k) + from + d;
                if constexpr (V == 8) *reinterpret_cast<uint2*>(c[w]) = *reinterpret_cast<const uint2*>(p);
                else c[w][0] = *reinterpret_cast<const uint32_t*>(p);
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float f = exp_of_byte((bytes >> (8 * w)) & 0xffu);
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const uint32_t lo = e4m3x2_to_f16x2(c[w][i / 4]), hi = e4m3x2_hi_to_f16x2(c[w][i / 4]);
                    x[w][i] = f16_lo(lo) * f;
                    x[w][i + 1] = f16_hi(lo) * f;
                    x[w][i + 2] = f16_lo(hi) * f;
                    x[w][i + 3] = f16_hi(hi) * f;
                }
            }
        } else {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint16_t* p = static_cast<const uint16_t*>(w ? a.pool_v : a.pool_k) + from + d;
                uint16_t c[V];
                load_run<uint16_t, V, true>(p, c);
#pragma unroll
                for (int i = 0; i < V; ++i) x[w][i] = bf16_to_f32(c[i]);
            }
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        T y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = E::put(x[w][i]);
        T* to = static_cast<T*>(w ? a.v : a.k) + token * (w ? a.v_stride : a.k_stride) + head * D + d;
        store_run<T, V, VEC>(to, y);
    }
}

template <int TYPE, int D, bool E4M3>
void launch_rows(bool write, bool vec, const RowsArgs& a, cudaStream_t s) {
    const int per = write ? 8 : 16 / static_cast<int>(sizeof(typename Elem<TYPE>::T));
    const long long threads = static_cast<long long>(a.n) * a.n_kv * (D / per);
    const long long blocks = (threads + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL) throw std::invalid_argument("KV rows: too many in one call");
    const dim3 grid(static_cast<unsigned>(blocks));
    auto kernel = write ? (vec ? kv_write_kernel<TYPE, D, E4M3, true> : kv_write_kernel<TYPE, D, E4M3, false>)
                        : (vec ? kv_read_kernel<TYPE, D, E4M3, true> : kv_read_kernel<TYPE, D, E4M3, false>);
    launch_dep(false, kernel, grid, dim3(kThreads), 0, s, a);
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
