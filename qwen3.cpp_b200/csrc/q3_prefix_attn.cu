// The shared prefix of q3_prefix_attn on tcgen05 tensor cores (sm_100a): the query rows of all
// sequences against one run of keys, so the prefix is read once for the batch.
//
// The rows of one KV head (query token x head of the group) are cut into tiles of 128, the prefix into
// tiles of 128 keys and those into splits, so that (heads x row tiles x splits) fills the GPU; each
// split leaves a part (max, sum, sums of p v) that join_kernel adds. A CTA keeps two streams going, so
// that the tensor cores work on one while the softmax of the other runs:
//   PAIR  more than 128 rows: two row tiles, each over all of the CTA's key tiles; K and V are brought
//         in once for both
//   SOLO  one row tile: one stream over the even key tiles, one over the odd ones (a part each)
// Per stream and key tile:
//   issuer   S = Q . K^T                  tcgen05.mma, M = N = 128, into TMEM
//   softmax  P = 2^(S c - m + kShift)      one thread a row; P replaces S in TMEM, as fp16 (e4m3 pool) or
//            as a bf16 pair hi + lo (bf16 pool)
//   issuer   O += P . V                   A from TMEM, V as it lies in shared memory (MN-major)
// O stays in TMEM. The running maximum moves only when a score passes it by more than 2^kGrow; then
// the row's O is read, scaled and written back (rare after the first tile).
//
// Four warps bring the tiles in: 16-byte loads one tile ahead, written in the operands' 128-byte
// swizzled layout. e4m3 codes become fp16 there, exactly, times 2^(byte - largest byte of the CTA's
// keys): exact down to 2^-15 of the largest row, below that to 2^-25 of its unit. One factor in front
// of the scores and one behind the sums then stand for all bytes.
//
// Warps: 0-3 and 4-7 softmax of stream 0 and 1, 8-11 loaders, 12 issuer. Every wait is bounded; one
// that gives up ends the CTA's loops and leaves NaN in its parts.
#include <algorithm>

#include "q3_paged_attn.cuh"
#include "q3_sm100.cuh"

namespace q3 {

namespace {

using namespace sm100;

constexpr int kRowTile = 128, kKeyTile = 128;
constexpr int kPagesPerTile = kKeyTile / kPageTokens;
constexpr int kMaxTiles = 512;      // key tiles of one CTA (the size of its list of good pages)
constexpr int kPrefixThreads = 416;
constexpr float kGrow = 6.0f;       // weights are at most 2^(kShift + kGrow) = 2^14
constexpr long long kBudget = 4000000000LL;  // cycles, about 2 s
constexpr int kPanel = 128 * 128;   // bytes of 64 columns of 128 rows
constexpr uint32_t kTmemCols = 512; // S of both streams, then O of both: 128 columns each

template <int D, bool PAIR>
struct Smem {
    static constexpr int kTile = D / 64 * kPanel;
    static constexpr int kStages = PAIR ? 2 : 3;  // of K, and of V
    static constexpr int kQ = 0;
    static constexpr int kK = (PAIR ? 2 : 1) * kTile;
    static constexpr int kV = kK + kStages * kTile;
    static constexpr int kBar = kV + kStages * kTile;
    static constexpr int kMask = kBar + 256;
    static constexpr int kBytes = kMask + kMaxTiles;
};

__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr, uint32_t panel_bytes) {
    uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFF) >> 4);
    d |= static_cast<uint64_t>((panel_bytes >> 4) & 0x3FFF) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

__device__ __forceinline__ void fence_smem_to_mma() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]: A's rows are TMEM lanes, two 16-bit values a column.
__device__ __forceinline__ void mma_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// fp16 2^e for e <= 0, twice.
__device__ __forceinline__ uint32_t half2_pow2(int e) {
    const uint32_t h = e >= -14 ? static_cast<uint32_t>(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
    return h | h << 16;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <int D, bool E4M3, bool PAIR>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_kernel(const PagedArgs a) {
    using L = Smem<D, PAIR>;
    constexpr int STAGES = L::kStages;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBar);
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;
    uint64_t* k_empty = bars + 4;
    uint64_t* v_full = bars + 7;
    uint64_t* v_empty = bars + 10;
    uint64_t* s_full = bars + 13;
    uint64_t* p_full = bars + 15;
    uint64_t* o_full = bars + 17;
    uint64_t* done = bars + 19;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* top_s = reinterpret_cast<int*>(tmem_slot + 2);  // largest byte of K, of V
    uint8_t* mask = sm + L::kMask;                       // a bit a good page of each key tile

    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.n_q * a.group;
    const int split = blockIdx.x, h = blockIdx.y;
    const int row_base = blockIdx.z * (PAIR ? 2 : 1) * kRowTile;
    const int all_tiles = (a.prefix_len + kKeyTile - 1) / kKeyTile;
    const int cta_splits = gridDim.x;
    const int tile0 = static_cast<int>(static_cast<long long>(all_tiles) * split / cta_splits);
    const int n_tiles = static_cast<int>(static_cast<long long>(all_tiles) * (split + 1) / cta_splits) - tile0;
    const int all_pages = (a.prefix_len + kPageTokens - 1) / kPageTokens;

    if ((smem_u32(sm) & 1023) != 0 || n_tiles > kMaxTiles) {
        // Not reached: the operands need a 1024-byte aligned base, the list of pages its length.
        for (int r = tid; r < (PAIR ? 2 : 1) * kRowTile && row_base + r < rows; r += kPrefixThreads) {
            const size_t part = PAIR ? split : split * 2;
            const float bad = __int_as_float(0x7fc00000);
            a.prefix_ml[(part * a.n_kv + h) * a.prefix_rows + row_base + r] = make_float2(bad, bad);
        }
        return;
    }
    if (tid == 0) {
        mbar_init(q_full, PAIR ? 8 : 4);
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(done, 1);
        *abort = 0;
        top_s[0] = top_s[1] = 0;
        mbar_fence_init();
    }
    for (int i = tid; i < n_tiles; i += kPrefixThreads) mask[i] = 0;
    if (warp == 12) tmem_alloc(tmem_slot, kTmemCols);
    __syncthreads();
    // The CTA's good pages and the largest bytes of its keys.
    for (int p = tid; p < n_tiles * kPagesPerTile; p += kPrefixThreads) {
        const int logical = tile0 * kPagesPerTile + p;
        const int page = logical < all_pages ? a.prefix_table[logical] : -1;
        if (page < 0 || page >= a.n_pages) continue;
        atomicOr(reinterpret_cast<unsigned*>(mask) + p / 32, 1u << (p % 32));
        if constexpr (E4M3) {
            const uint4* e = reinterpret_cast<const uint4*>(
                a.exps + (static_cast<size_t>(page) * a.n_kv + h) * kPageTokens * 2);
            const uint32_t* e4 = reinterpret_cast<const uint32_t*>(e);
            const int n = min(kPageTokens, a.prefix_len - logical * kPageTokens);
            uint32_t kt = 0, vt = 0;
#pragma unroll
            for (int i = 0; i < kPageTokens / 2; ++i) {
                const uint32_t x = __ldg(e4 + i);
                if (2 * i < n) {
                    kt = max(kt, x & 0xffu);
                    vt = max(vt, x >> 8 & 0xffu);
                }
                if (2 * i + 1 < n) {
                    kt = max(kt, x >> 16 & 0xffu);
                    vt = max(vt, x >> 24);
                }
            }
            atomicMax(&top_s[0], static_cast<int>(kt));
            atomicMax(&top_s[1], static_cast<int>(vt));
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int top_k = top_s[0], top_v = top_s[1];
    // Steps of a stream: its key tiles.
    auto steps_of = [&](int s) { return PAIR ? n_tiles : (n_tiles + 1 - s) / 2; };

    if (warp == 12) {
        if (lane == 0) {
            // ------------------------------------------------------------ issuer
            const uint32_t idesc_s = E4M3 ? idesc_f16_f32(kRowTile, kKeyTile) : idesc_bf16_f32(kRowTile, kKeyTile);
            const uint32_t idesc_pv = (E4M3 ? idesc_f16_f32(kRowTile, D) : idesc_bf16_f32(kRowTile, D)) |
                                      (1u << 16);  // B MN-major
            bool ok = mbar_wait(q_full, 0, kBudget, abort);
            auto scores = [&](int s, int i) {
                const int j = PAIR ? i : 2 * i + s, st = j % STAGES;
                if (!mbar_wait(&k_full[st], (j / STAGES) & 1, kBudget, abort)) return false;
                tc_fence_after();
                const uint32_t q_addr = smem_u32(sm + L::kQ + (PAIR ? s * L::kTile : 0));
                const uint32_t k_addr = smem_u32(sm + L::kK + st * L::kTile);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    mma_bf16(tmem + s * 128, desc_k_sw128(q_addr + (kk >> 2) * kPanel) + 2 * (kk & 3),
                             desc_k_sw128(k_addr + (kk >> 2) * kPanel) + 2 * (kk & 3), idesc_s, kk > 0);
                }
                mma_commit(&s_full[s]);
                if (!PAIR || s == 1) mma_commit(&k_empty[st]);
                return true;
            };
            for (int s = 0; s < 2 && ok; ++s) {
                if (steps_of(s) > 0) ok = scores(s, 0);
            }
            const int most = steps_of(0);
            for (int i = 0; ok && i < most; ++i) {
                for (int s = 0; s < 2 && ok; ++s) {
                    if (i >= steps_of(s)) continue;
                    const int j = PAIR ? i : 2 * i + s, st = j % STAGES;
                    ok = mbar_wait(&p_full[s], i & 1, kBudget, abort) &&
                         mbar_wait(&v_full[st], (j / STAGES) & 1, kBudget, abort);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t v_addr = smem_u32(sm + L::kV + st * L::kTile);
                    const uint32_t o = tmem + 256 + s * 128, p = tmem + s * 128;
#pragma unroll
                    for (int kk = 0; kk < kKeyTile / 16; ++kk) {
                        const uint64_t v = desc_mn_sw128(v_addr + kk * 16 * 128, kPanel);
                        if constexpr (E4M3) {
                            mma_a_tmem(o, p + kk * 8, v, idesc_pv, i > 0 || kk > 0);
                        } else {
                            const uint32_t at = p + (kk >> 1) * 32 + (kk & 1) * 8;
                            mma_a_tmem(o, at, v, idesc_pv, i > 0 || kk > 0);
                            mma_a_tmem(o, at + 16, v, idesc_pv, 1);
                        }
                    }
                    if (!PAIR || s == 1) mma_commit(&v_empty[st]);
                    if (i + 1 < steps_of(s)) ok = scores(s, i + 1);
                    else mma_commit(&o_full[s]);
                }
            }
            if (!ok) *abort = 1;
            // Nothing is in flight when the CTA ends.
            mma_commit(done);
            if (!mbar_wait(done, 0, kBudget, abort)) {
                const long long t0 = clock64();
                while (!mbar_try_wait(done, 0) && clock64() - t0 < kBudget) {}
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ---------------------------------------------------------------- loaders
        constexpr int ROW = E4M3 ? D : 2 * D;      // bytes of a pool row
        constexpr int CHUNKS = ROW / 16;           // 16-byte pieces of a row
        constexpr int LANES = 128 / CHUNKS;        // rows that one round of loads covers
        constexpr int LOADS = kKeyTile / LANES;    // rounds of a tile
        constexpr int BATCH = LOADS < 8 ? LOADS : 8;
        constexpr int BATCHES = LOADS / BATCH;     // of a tile
        const int lt = tid - 256, c = lt % CHUNKS, r0 = lt / CHUNKS;
        const int total = n_tiles * 2 * BATCHES;   // K 0, V 0, K 1, V 1, ...
        uint4 raw[2][BATCH];
        uint32_t ex[2][BATCH];
        auto load = [&](int n, uint4 (&x)[BATCH], uint32_t (&e)[BATCH]) {
            const int j = n / (2 * BATCHES), kind = n / BATCHES & 1, part = n % BATCHES;
            const uint8_t* base = static_cast<const uint8_t*>(kind ? a.v : a.k);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = r0 + (part * BATCH + i) * LANES;
                const int key = (tile0 + j) * kKeyTile + r;
                x[i] = make_uint4(0, 0, 0, 0);
                e[i] = 0;
                if (key >= a.prefix_len) continue;
                const int page = __ldg(a.prefix_table + key / kPageTokens);
                if (page < 0 || page >= a.n_pages) continue;
                const size_t row = (static_cast<size_t>(page) * a.n_kv + h) * kPageTokens + key % kPageTokens;
                x[i] = *reinterpret_cast<const uint4*>(base + row * ROW + c * 16);
                if constexpr (E4M3) e[i] = a.exps[row * 2 + kind];
            }
        };
        auto store = [&](int n, const uint4 (&x)[BATCH], const uint32_t (&e)[BATCH]) {
            const int j = n / (2 * BATCHES), kind = n / BATCHES & 1, part = n % BATCHES;
            const int st = j % STAGES;
            uint8_t* to = sm + (kind ? L::kV : L::kK) + st * L::kTile;
            if (part == 0 && !mbar_wait_warp(kind ? &v_empty[st] : &k_empty[st], ((j / STAGES) & 1) ^ 1,
                                             kBudget, abort)) {
                return false;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = r0 + (part * BATCH + i) * LANES;
                if constexpr (E4M3) {
                    const uint32_t f = half2_pow2(static_cast<int>(e[i]) - (kind ? top_v : top_k));
                    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                    uint32_t y[8];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        y[2 * q] = mul_half2(e4m3x2_to_f16x2(w[q]), f);
                        y[2 * q + 1] = mul_half2(e4m3x2_hi_to_f16x2(w[q]), f);
                    }
                    uint8_t* row = to + (c >> 2) * kPanel + r * 128;
                    const uint4 lo = make_uint4(y[0], y[1], y[2], y[3]), hi = make_uint4(y[4], y[5], y[6], y[7]);
                    // The pieces of one row go to different banks: the second panel's halves swapped.
                    const int first = (c >> 2) & 1;
                    *reinterpret_cast<uint4*>(row + ((((c & 3) * 2 + first) ^ (r & 7)) * 16)) = first ? hi : lo;
                    *reinterpret_cast<uint4*>(row + ((((c & 3) * 2 + 1 - first) ^ (r & 7)) * 16)) = first ? lo : hi;
                } else {
                    *reinterpret_cast<uint4*>(to + (c >> 3) * kPanel + r * 128 + (((c & 7) ^ (r & 7)) * 16)) = x[i];
                }
            }
            if (part == BATCHES - 1) {
                fence_smem_to_mma();
                __syncwarp();
                if (lane == 0) mbar_arrive(kind ? &v_full[st] : &k_full[st]);
            }
            return true;
        };
        load(0, raw[0], ex[0]);
        bool ok = true;
        for (int n = 0; ok && n < total; n += 2) {  // total is even
            load(n + 1, raw[1], ex[1]);
            ok = store(n, raw[0], ex[0]);
            if (ok && n + 2 < total) load(n + 2, raw[0], ex[0]);
            ok = ok && store(n + 1, raw[1], ex[1]);
        }
        if (!ok) *abort = 1;
    } else {
        // ---------------------------------------------------------------- softmax
        const int s = warp >> 2, r = (warp & 3) * 32 + lane;
        const int row = row_base + (PAIR ? s * kRowTile : 0) + r;
        const bool live = row < rows;
        float c = 1.4426950408889634f / sqrtf(static_cast<float>(D));
        {
            // This row of Q into the operand, scaled by a power of two for fp16.
            const uint16_t* q = static_cast<const uint16_t*>(a.q) +
                                (live ? row / a.group * a.q_stride + (h * a.group + row % a.group) * D : 0);
            uint4 x[D / 8];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                x[i] = live ? reinterpret_cast<const uint4*>(q)[i] : make_uint4(0, 0, 0, 0);
            }
            if constexpr (E4M3) {
                uint32_t* w = reinterpret_cast<uint32_t*>(x);
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 2; ++i) {
                    big = max3(big, fabsf(a.f16 ? f16_lo(w[i]) : bf16_lo(w[i])),
                               fabsf(a.f16 ? f16_hi(w[i]) : bf16_hi(w[i])));
                }
                int e = 0;
                if (big > 0.0f && big < INFINITY) {
                    e = min(13 + 127 - static_cast<int>(__float_as_uint(big) >> 23), 126);
                }
                const float f = pow2(e);
#pragma unroll
                for (int i = 0; i < D / 2; ++i) {
                    w[i] = pack2_out((a.f16 ? f16_lo(w[i]) : bf16_lo(w[i])) * f,
                                     (a.f16 ? f16_hi(w[i]) : bf16_hi(w[i])) * f, 1);
                }
                // Kept a normal number: a masked score is -infinity times it.
                c = fminf(fmaxf(c * pow2(-e) * exp_of_byte(static_cast<uint32_t>(top_k)), 1e-37f), 1e37f);
            }
            if (PAIR || s == 0) {
                uint8_t* to = sm + L::kQ + (PAIR ? s * L::kTile : 0) + r * 128;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    *reinterpret_cast<uint4*>(to + (i >> 3) * kPanel + (((i & 7) ^ (r & 7)) * 16)) = x[i];
                }
                fence_smem_to_mma();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
        }
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + s * 128, o_at = tmem + lanes + 256 + s * 128;
        float m = -INFINITY, neg = kShift;
        float2 l2 = make_float2(0.0f, 0.0f);
        const int steps = steps_of(s);
        bool ok = true;
        for (int i = 0; i < steps; ++i) {
            const int j = PAIR ? i : 2 * i + s;
            if (!mbar_wait_warp(&s_full[s], i & 1, kBudget, abort)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const bool full = mask[j] == 0xff && (tile0 + j + 1) * kKeyTile <= a.prefix_len;
            // A key that is not there: its bit, and its place before the end.
            auto there = [&](int k) {
                return (mask[j] >> (k / kPageTokens) & 1) && (tile0 + j) * kKeyTile + k < a.prefix_len;
            };
            float top = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float x[32];
                tmem_ld32(s_at + q * 32, x);
                if (!full) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = there(q * 32 + k) ? x[k] : -INFINITY;
                }
#pragma unroll
                for (int k = 0; k < 32; k += 2) top = max3(top, x[k], x[k + 1]);
            }
            if (__any_sync(0xffffffffu, top * c > m + kGrow)) {
                const float m_new = fmaxf(m, top * c);
                const float f = m_new == m ? 1.0f : ex2(m - m_new);
                m = m_new;
                neg = kShift - (m_new == -INFINITY ? 0.0f : m_new);
                l2.x *= f;
                l2.y *= f;
                if (i > 0) {  // the products before this tile's scores are done: O is still
#pragma unroll 1
                    for (int q = 0; q < D / 32; ++q) {
                        float x[32];
                        uint32_t y[32];
                        tmem_ld32(o_at + q * 32, x);
#pragma unroll
                        for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(x[k] * f);
                        tmem_st32(o_at + q * 32, y);
                    }
                    tmem_st_wait();
                }
            }
            const float2 c2 = make_float2(c, c), n2 = make_float2(neg, neg);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t y[32];  // fp16: 64 keys; bf16: 32 keys at a time, hi and lo
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int k0 = (half * 2 + q) * 32;
                    float x[32];
                    tmem_ld32(s_at + k0, x);
                    if (!full) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) x[k] = there(k0 + k) ? x[k] : -INFINITY;
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float2 p = ffma2(make_float2(x[k], x[k + 1]), c2, n2);
                        p.x = ex2(p.x);
                        p.y = ex2(p.y);
                        l2 = fadd2(l2, p);
                        if constexpr (E4M3) {
                            y[q * 16 + k / 2] = pack2_out(p.x, p.y, 1);
                        } else {
                            const uint32_t w = pack2_bf16(p.x, p.y);
                            y[k / 2] = w;
                            y[16 + k / 2] = pack2_bf16(p.x - bf16_lo(w), p.y - bf16_hi(w));
                        }
                    }
                    if constexpr (!E4M3) tmem_st32(s_at + k0, y);
                }
                if constexpr (E4M3) tmem_st32(s_at + half * 32, y);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[s]);
        }
        if (ok && steps > 0) ok = mbar_wait_warp(&o_full[s], 0, kBudget, abort);
        if (!ok) *abort = 1;
        const size_t part = PAIR ? split : split * 2 + s;
        const size_t at = (part * a.n_kv + h) * a.prefix_rows + row;
        const float f_v = E4M3 ? exp_of_byte(static_cast<uint32_t>(top_v)) : 1.0f;
        tc_fence_after();
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
            float x[32];
            if (ok && steps > 0) {
                tmem_ld32(o_at + q * 32, x);
            } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) x[k] = 0.0f;
            }
            if (live) {
                float4* to = reinterpret_cast<float4*>(a.prefix_o + at * D + q * 32);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    to[k] = make_float4(x[4 * k] * f_v, x[4 * k + 1] * f_v, x[4 * k + 2] * f_v, x[4 * k + 3] * f_v);
                }
            }
        }
        if (live) {
            const float bad = __int_as_float(0x7fc00000);
            a.prefix_ml[at] = ok ? make_float2(m, l2.x + l2.y) : make_float2(bad, bad);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <int D, bool E4M3, bool PAIR>
void launch(const PagedArgs& a, cudaStream_t s) {
    const int rows = a.n_q * a.group, tile = (PAIR ? 2 : 1) * kRowTile;
    const dim3 grid(PAIR ? a.prefix_splits : a.prefix_splits / 2, a.n_kv, (rows + tile - 1) / tile);
    constexpr int bytes = Smem<D, PAIR>::kBytes;
    Q3_CUDA(cudaFuncSetAttribute(prefix_kernel<D, E4M3, PAIR>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    launch_dep(false, prefix_kernel<D, E4M3, PAIR>, grid, dim3(kPrefixThreads), bytes, s, a);
}

template <int D>
void launch(const PagedArgs& a, bool e4m3, cudaStream_t s) {
    const bool pair = a.n_q * a.group > kRowTile;
    if (e4m3) pair ? launch<D, true, true>(a, s) : launch<D, true, false>(a, s);
    else pair ? launch<D, false, true>(a, s) : launch<D, false, false>(a, s);
}

}  // namespace

// Parts per row. A CTA's time is about (its key tiles + 3), 3 for its start and end; the splits make the
// sum over the waves of 148 CTAs least. PAIR CTAs leave one part, SOLO ones two.
int prefix_splits(int n_kv, int rows, int prefix_len) {
    if (prefix_len <= 0 || rows <= 0) return 0;
    const bool pair = rows > kRowTile;
    const long long base = static_cast<long long>(n_kv) * (pair ? (rows + 2 * kRowTile - 1) / (2 * kRowTile) : 1);
    const long long tiles = (static_cast<long long>(prefix_len) + kKeyTile - 1) / kKeyTile;
    const long long least = (tiles + kMaxTiles - 1) / kMaxTiles;
    long long best = least, best_cost = -1;
    for (long long n = least; n <= std::max(least, std::min(tiles, 64LL)); ++n) {
        const long long waves = (base * n + 147) / 148, each = (tiles + n - 1) / n;
        const long long cost = waves * ((pair ? 2 : 1) * each + 3);
        if (best_cost < 0 || cost < best_cost) {
            best = n;
            best_cost = cost;
        }
    }
    return static_cast<int>(pair ? best : 2 * best);
}

void launch_prefix_attention(const PagedArgs& a, int head_dim, bool e4m3, cudaStream_t s) {
    if (head_dim == 64) launch<64>(a, e4m3, s);
    else launch<128>(a, e4m3, s);
}

}  // namespace q3
