// The shared prefix of q3_prefix_attn on tcgen05 tensor cores (sm_100a): the query rows of all
// sequences against one run of keys, so the prefix is read once for the batch.
//
// The rows of one KV head (query token x head of the group) are cut into tiles of 128, the prefix into
// tiles of 128 keys and those into splits, so that (heads x row tiles x splits) fills the GPU; each
// split leaves a part (max, sum, sums of p v) that join_kernel adds. A CTA keeps two streams going, so
// that the tensor cores work on one while the softmax of the other runs:
//   PAIR  more than 128 rows: two row tiles, each over all of the CTA's key tiles; K and V are brought
//         in once for both
//   SOLO  one row tile: one stream over the even key tiles, one over the odd ones, added at the end
// Per stream and key tile:
//   issuer   S = Q . K^T                  tcgen05.mma, M = N = 128, into TMEM
//   softmax  P = 2^(S c - m + kShift)      one thread a row; P replaces S in TMEM, as fp16 (e4m3 pool) or
//            as a bf16 pair hi + lo (bf16 pool)
//   issuer   O += P . V                   A from TMEM, V as it lies in shared memory (MN-major)
// O stays in TMEM. The running maximum moves only when a score passes it by more than 2^kGrow; then
// the row's O is read, scaled and written back (rare after the first tile).
//
// Four warps bring the tiles in by cp.async, ahead of their use, into the operands' 128-byte swizzled
// layout: bf16 directly; e4m3 codes by way of a ring of raw tiles, from which they become fp16
// times 2^(byte - largest byte of the CTA's keys + kLift). kLift takes the largest code to 57344, near fp16's
// end: a row is exact where its power of two is 2^-22 or more of the CTA's largest, else rounded to 2^-32 of
// that. One factor in front of the scores and one behind the sums then stand for all bytes.
//
// Warps: 0-3 and 4-7 softmax of stream 0 and 1 (a row's 128 scores stay in registers, hence the uneven
// split of the registers), 8-11 loaders, 12 issuer. Every wait is bounded; one that gives up ends the
// CTA's loops and leaves NaN in its parts.
//
// Bound by 4 * D operations a row, head and key for many rows, by latency for few. 427 rows of 32 heads,
// 8 KV heads of 128, 32768 keys (e4m3): 229 GFLOP in 240 us alone, launch by launch (267 on another B200), 0.95
// PFLOP/s, the tensor pipe and the exponentials' 41% busy each, shared memory about 68% (scores read 128 bytes
// a cycle, the loaders write the raw and the converted tiles), the power limit reached in a row of calls. 8192
// keys for 64 rows of 16 heads: 17 us. In a bf16 pool, with three products where e4m3 has two, the whole call
// over 427 rows and 32768 keys takes 332 us against 283.
#include <algorithm>

#include "q3_paged_attn.cuh"
#include "q3_sm100.cuh"

namespace q3 {

namespace {

using namespace sm100;

constexpr int kRowTile = 128, kKeyTile = 128;
constexpr int kPagesPerTile = kKeyTile / kPageTokens;
constexpr int kMaxTiles = 512;      // key tiles of one CTA (the size of its list of good pages)
constexpr int kPrefixThreads = 512;
constexpr int kManyRegs = 192, kFewRegs = 64;  // 8 warps each: 512 threads are launched with 128
constexpr int kLift = 7;            // see above: 448 * 2^7 is below 65504
constexpr float kGrow = 6.0f;       // weights are at most 2^(kShift + kGrow) = 2^14
constexpr long long kBudget = 4000000000LL;  // cycles, about 2 s
constexpr int kPanel = 128 * 128;   // bytes of 64 columns of 128 rows
constexpr uint32_t kTmemCols = 512; // S of both streams, then O of both: 128 columns each

template <int D, bool E4M3, bool PAIR>
struct Smem {
    static constexpr int kTile = D / 64 * kPanel;
    static constexpr int kSlots = E4M3 ? (PAIR ? 3 : 4) : (PAIR ? 5 : 6);  // K and V tiles, in turn
    static constexpr int kRaw = E4M3 ? 4 : 0;                              // raw tiles on their way
    static constexpr int kQ = 0;
    static constexpr int kKv = (PAIR ? 2 : 1) * kTile;
    static constexpr int kRing = kKv + kSlots * kTile;
    static constexpr int kExps = kRing + kRaw * kTile / 2;  // [4 tiles][128 keys][2] bytes
    static constexpr int kScale = kExps + (E4M3 ? 4 * kKeyTile * 2 : 0);  // [4 warps][32 keys] fp16 pairs
    static constexpr int kBar = kScale + (E4M3 ? kKeyTile * 4 : 0);
    static constexpr int kMask = kBar + 256;
    // After the last product the sums of the 8 softmax warps take the tiles' room.
    static_assert(kBar - kKv >= 8 * 32 * D * 4, "room for the sums");
    static constexpr int kBytes = kMask + kMaxTiles;
    static_assert(kBytes <= 232448, "shared memory of a CTA");
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

__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}

// The tensor-core instructions of the issuing thread, which is chosen by elect.sync. (Issued by lane 0 of
// an ordinary branch an MMA takes about 95 cycles to issue, more than its 64 in the pipe.)
// D[tmem] (+)= A[smem] * B[smem]^T
__device__ __forceinline__ void issue_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: A's rows are TMEM lanes, two 16-bit values a column.
__device__ __forceinline__ void issue_mma_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                                 uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void issue_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
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

// 64 consecutive columns of this thread's TMEM lane. The load and its wait are one statement, so no use
// of the values can move above the wait.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
          "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
          "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
          "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
          "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
          "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// Registers a thread of this warpgroup: the sum over the block's is what it was launched with.
template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// The softmax warps' own barrier.
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// The same, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// fp16 2^e for e <= kLift, twice.
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
    using L = Smem<D, E4M3, PAIR>;
    constexpr int SLOTS = L::kSlots;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBar);
    uint64_t* q_full = bars;
    uint64_t* full = bars + 1;    // [SLOTS]
    uint64_t* empty = bars + 7;   // [SLOTS]
    uint64_t* s_full = bars + 13;
    uint64_t* p_full = bars + 15;  // [stream][half of the keys]
    uint64_t* o_full = bars + 19;
    uint64_t* done = bars + 21;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* top_s = reinterpret_cast<int*>(tmem_slot + 2);  // largest byte of K, of V
    uint8_t* mask = sm + L::kMask;                       // a bit a good page of each key tile

    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.n_q * a.group;
    const int split = blockIdx.x, h = blockIdx.y;
    const int row_base = blockIdx.z * (PAIR ? 2 : 1) * kRowTile;
    const int all_tiles = (a.prefix_len + kKeyTile - 1) / kKeyTile;
    const int tile0 = static_cast<int>(static_cast<long long>(all_tiles) * split / gridDim.x);
    const int n_tiles = static_cast<int>(static_cast<long long>(all_tiles) * (split + 1) / gridDim.x) - tile0;
    const int all_pages = (a.prefix_len + kPageTokens - 1) / kPageTokens;
    const size_t part = (static_cast<size_t>(split) * a.n_kv + h) * a.prefix_rows;

    if ((smem_u32(sm) & 1023) != 0 || n_tiles > kMaxTiles) {
        // Not reached: the operands need a 1024-byte aligned base, the list of pages its length.
        const float bad = __int_as_float(0x7fc00000);
        for (int r = tid; r < (PAIR ? 2 : 1) * kRowTile && row_base + r < rows; r += kPrefixThreads) {
            a.prefix_ml[part + row_base + r] = make_float2(bad, bad);
        }
        return;
    }

    // ---------------------------------------------------------------- loaders: tiles on their way
    // Loader warp w brings the 32 keys of pages 2w, 2w + 1 of each tile; operations are K 0, V 0, K 1, ...
    constexpr int ROW = E4M3 ? D : 2 * D;                // bytes of a pool row
    constexpr int CHUNKS = ROW / 16;                     // 16-byte pieces of a row
    constexpr int LOADS = CHUNKS;                        // pieces of 32 rows, a lane
    // Lane's place in load i: for e4m3 eight rows of four pieces (of one operand panel), so that the
    // converted pieces of two neighbouring rows fall into all banks; else rows one after the other.
    constexpr int PANELS = E4M3 ? D / 64 : 1;
    auto place = [&](int i, int& r, int& c) {
        if constexpr (E4M3) {
            r = i / PANELS * 8 + lane / 4;
            c = i % PANELS * 4 + lane % 4;
        } else {
            const int x = i * 32 + lane;
            r = x / CHUNKS;
            c = x % CHUNKS;
        }
    };
    // Its place in a raw tile: odd rows' panels swapped, so that two rows' reads fall into all banks.
    auto raw_at = [&](int key, int c) { return key * D + (PANELS == 2 ? c ^ (key & 1) * 4 : c) * 16; };
    const int lw = warp & 3;
    int ids = -1;  // lane: page 2w + (lane & 1) of tile (lane / 2) of the 16 looked up
    auto look_up_tiles = [&](int j) {
        const int t = j + lane / 2;
        const int logical = (tile0 + t) * kPagesPerTile + 2 * lw + (lane & 1);
        ids = t < n_tiles && logical < all_pages ? __ldg(a.prefix_table + logical) : -1;
    };
    auto issue = [&](int n, uint8_t* to) {  // in order
        const int j = n >> 1, kind = n & 1;
        if (!kind && (j & 15) == 0 && j > 0) look_up_tiles(j);
        const uint8_t* base = static_cast<const uint8_t*>(kind ? a.v : a.k);
        const int left = a.prefix_len - (tile0 + j) * kKeyTile - lw * 32;  // keys of this warp's 32 that exist
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int page = __shfl_sync(0xffffffffu, ids, (j & 15) * 2 + half);
            const bool in = page >= 0 && page < a.n_pages;
            const size_t row0 = (static_cast<size_t>(in ? page : 0) * a.n_kv + h) * kPageTokens;
            const uint8_t* from = base + row0 * ROW;
#pragma unroll
            for (int i = 0; i < LOADS / 2; ++i) {
                int rr, c;
                place(half * (LOADS / 2) + i, rr, c);
                const int key = lw * 32 + rr;
                uint8_t* dst = E4M3 ? to + raw_at(key, c)
                                    : to + (c >> 3) * kPanel + key * 128 + (((c & 7) ^ (key & 7)) * 16);
                // A key that is not there becomes zeros.
                const int bytes = in && rr < left ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)),
                             "l"(from + (rr - half * 16) * ROW + c * 16), "r"(bytes)
                             : "memory");
            }
            if (E4M3 && !kind && lane < 8) {
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                                 smem_u32(sm + L::kExps + ((j & 3) * kKeyTile + lw * 32 + half * 16) * 2 + lane * 4)),
                             "l"(a.exps + row0 * 2 + lane * 4), "r"(in ? 4 : 0)
                             : "memory");
            }
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    auto raw = [&](int n) { return sm + L::kRing + n % (L::kRaw ? L::kRaw : 1) * (L::kTile / 2); };
    const int ops = 2 * n_tiles;
    const bool is_loader = warp >= 8 && warp < 12;

    // The CTA's pages and the bytes of their keys: a thread a page. The first are on their way before anything
    // waits, the loaders' behind their first tiles (64 x 8192: 32.5 us, 33.4 with all of them after the set-up).
    const int n_pages = min(n_tiles * kPagesPerTile, all_pages - tile0 * kPagesPerTile);
    struct Look {
        bool in;
        uint32_t w[E4M3 ? kPageTokens / 2 : 1];
    };
    auto look_up = [&](int p, int page) {
        Look x{};
        x.in = p < n_pages && page >= 0 && page < a.n_pages;
        if (E4M3 && x.in) {
            const uint32_t* e = reinterpret_cast<const uint32_t*>(
                a.exps + (static_cast<size_t>(page) * a.n_kv + h) * kPageTokens * 2);
#pragma unroll
            for (int i = 0; i < kPageTokens / 2; ++i) x.w[E4M3 ? i : 0] = __ldg(e + i);
        }
        return x;
    };
    auto page_of = [&](int p) { return p < n_pages ? __ldg(a.prefix_table + tile0 * kPagesPerTile + p) : -1; };
    const int first_page = page_of(tid);
    if (is_loader) look_up_tiles(0);
    Look mine{};
    if (!E4M3 || !is_loader) mine = look_up(tid, first_page);
    if (E4M3 && is_loader) {
#pragma unroll
        for (int n = 0; n < L::kRaw - 1; ++n) {
            if (n < ops) issue(n, raw(n));
            commit();
        }
        mine = look_up(tid, first_page);
    }
    // ---------------------------------------------------------------- softmax: the rows of Q on their way
    // Whole rows, Q_LANES lanes each, into their places in the operand (a thread reading its own row from
    // global memory touches 32 lines an instruction: 2 us for the CTA).
    constexpr int Q_LANES = D / 8, Q_ROWS = 32 / Q_LANES;
    const int s = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const int tile_row = row_base + (PAIR ? s * kRowTile : 0);
    const int row = tile_row + r;
    const bool live = warp < 8 && row < rows;
    uint8_t* q_tile = sm + L::kQ + (PAIR ? s * L::kTile : 0);
    if (warp < 8) {
        const int piece = lane % Q_LANES;
        // SOLO: the two streams' warps bring half of the one tile's rows each.
        const int first = (warp & 3) * 32 + (PAIR ? 0 : s * 16), n_rows = PAIR ? 32 : 16;
#pragma unroll
        for (int i = 0; i < n_rows; i += Q_ROWS) {
            const int qr = first + i + lane / Q_LANES, token = token_of(a, tile_row + qr);
            const bool in = tile_row + qr < rows;
            const uint16_t* from = static_cast<const uint16_t*>(a.q) + piece * 8 +
                                   (in ? token * a.q_stride + (h * a.group + tile_row + qr - token * a.group) * D : 0);
            uint8_t* to = q_tile + qr * 128 + (piece >> 3) * kPanel + (((piece & 7) ^ (qr & 7)) * 16);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(in ? 16 : 0)
                         : "memory");
        }
        commit();
    }

    if (tid == 0) {
        mbar_init(q_full, PAIR ? 8 : 4);
        for (int i = 0; i < SLOTS; ++i) {
            mbar_init(&full[i], 4);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(done, 1);
        *abort = 0;
        top_s[0] = top_s[1] = 0;
        mbar_fence_init();
    }
    if (warp == 12) tmem_alloc(tmem_slot, kTmemCols);
    __syncthreads();
    for (int p0 = warp * 32; p0 < n_pages; p0 += kPrefixThreads) {
        if (p0 != warp * 32) mine = look_up(p0 + lane, page_of(p0 + lane));
        const unsigned in = __ballot_sync(0xffffffffu, mine.in);
        if (lane == 0) reinterpret_cast<unsigned*>(mask)[p0 / 32] = in;
        if constexpr (E4M3) {
            const int n = a.prefix_len - (tile0 * kPagesPerTile + p0 + lane) * kPageTokens;  // the page's keys
            uint32_t kt = 0, vt = 0;
#pragma unroll
            for (int i = 0; i < kPageTokens / 2; ++i) {
                if (2 * i < n) {
                    kt = max(kt, mine.w[i] & 0xffu);
                    vt = max(vt, mine.w[i] >> 8 & 0xffu);
                }
                if (2 * i + 1 < n) {
                    kt = max(kt, mine.w[i] >> 16 & 0xffu);
                    vt = max(vt, mine.w[i] >> 24);
                }
            }
            // One of 32 lanes: same-address atomics of all would go one after the other.
            kt = __reduce_max_sync(0xffffffffu, kt);
            vt = __reduce_max_sync(0xffffffffu, vt);
            if (lane == 0) {
                atomicMax(&top_s[0], static_cast<int>(kt));
                atomicMax(&top_s[1], static_cast<int>(vt));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int top_k = top_s[0], top_v = top_s[1];
    // Steps of a stream: its key tiles.
    auto steps_of = [&](int s) { return PAIR ? n_tiles : (n_tiles + 1 - s) / 2; };

    if (warp >= 12) {
        fewer_registers<kFewRegs>();
        if (warp == 12 && elect_one()) {
            // ------------------------------------------------------------ issuer
            const uint32_t idesc_s = E4M3 ? idesc_f16_f32(kRowTile, kKeyTile) : idesc_bf16_f32(kRowTile, kKeyTile);
            const uint32_t idesc_pv = (E4M3 ? idesc_f16_f32(kRowTile, D) : idesc_bf16_f32(kRowTile, D)) |
                                      (1u << 16);  // B MN-major
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                return mbar_wait(bar, parity, kBudget, abort);
            };
            bool ok = wait(q_full, 0);
            auto scores = [&](int s, int i) {
                const int n = 2 * (PAIR ? i : 2 * i + s), slot = n % SLOTS;
                if (!wait(&full[slot], (n / SLOTS) & 1)) return false;
                tc_fence_after();
                const uint64_t qd = desc_k_sw128(smem_u32(sm + L::kQ + (PAIR ? s * L::kTile : 0)));
                const uint64_t kd = desc_k_sw128(smem_u32(sm + L::kKv + slot * L::kTile));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint64_t at = ((kk >> 2) * kPanel >> 4) + 2 * (kk & 3);
                    issue_mma(tmem + s * 128, qd + at, kd + at, idesc_s, kk > 0);
                }
                issue_commit(&s_full[s]);
                if (!PAIR || s == 1) issue_commit(&empty[slot]);
                return true;
            };
            for (int s = 0; s < 2 && ok; ++s) {
                if (steps_of(s) > 0) ok = scores(s, 0);
            }
            const int most = steps_of(0);
            for (int i = 0; ok && i < most; ++i) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!ok || i >= steps_of(s)) continue;
                    const int n = 2 * (PAIR ? i : 2 * i + s) + 1, slot = n % SLOTS;
                    ok = wait(&full[slot], (n / SLOTS) & 1) && wait(&p_full[2 * s], i & 1);
                    if (!ok) continue;
                    tc_fence_after();
                    const uint64_t vd = desc_mn_sw128(smem_u32(sm + L::kKv + slot * L::kTile), kPanel);
                    const uint32_t o = tmem + 256 + s * 128, p = tmem + s * 128;
                    auto product = [&](int kk) {
                        const uint64_t v = vd + kk * (16 * 128 >> 4);
                        issue_mma_a_tmem(o, p + kk * 8, v, idesc_pv, i > 0 || kk > 0);
                        if constexpr (!E4M3) issue_mma_a_tmem(o, p + 64 + kk * 8, v, idesc_pv, 1);
                    };
#pragma unroll
                    for (int kk = 0; kk < kKeyTile / 32; ++kk) product(kk);
                    ok = wait(&p_full[2 * s + 1], i & 1);
                    if (!ok) continue;
                    tc_fence_after();
#pragma unroll
                    for (int kk = kKeyTile / 32; kk < kKeyTile / 16; ++kk) product(kk);
                    if (!PAIR || s == 1) issue_commit(&empty[slot]);
                    if (i + 1 < steps_of(s)) ok = scores(s, i + 1);
                    else issue_commit(&o_full[s]);
                }
            }
            if (!ok) *abort = 1;
            // Nothing is in flight when the CTA ends.
            issue_commit(done);
            if (!wait(done, 0)) {
                const long long t0 = clock64();
                while (!mbar_try_wait(done, 0) && clock64() - t0 < kBudget) {}
            }
        }
        __syncwarp();
    } else if (is_loader) {
        // ---------------------------------------------------------------- loaders
        fewer_registers<kFewRegs>();
        bool ok = true;
        if constexpr (E4M3) {
            uint32_t* scale = reinterpret_cast<uint32_t*>(sm + L::kScale) + lw * 32;
            for (int n = 0; ok && n < ops; ++n) {
                const int j = n >> 1, kind = n & 1, slot = n % SLOTS;
                asm volatile("cp.async.wait_group %0;" ::"n"(L::kRaw - 2) : "memory");
                __syncwarp();
                // A lane a key: its power of two relative to the largest.
                const int e = sm[L::kExps + ((j & 3) * kKeyTile + lw * 32 + lane) * 2 + kind];
                scale[lane] = half2_pow2(min(e - (kind ? top_v : top_k), 0) + kLift);
                if (n + L::kRaw - 1 < ops) issue(n + L::kRaw - 1, raw(n + L::kRaw - 1));
                commit();
                if (!mbar_wait_warp(&empty[slot], ((n / SLOTS) & 1) ^ 1, kBudget, abort)) {
                    ok = false;
                    break;
                }
                __syncwarp();
                uint8_t* to = sm + L::kKv + slot * L::kTile;
                const uint8_t* from = raw(n);
                // All reads first: the compiler does not move one above a write.
                uint4 w[LOADS];
                uint32_t f[LOADS];
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    int rr, c;
                    place(i, rr, c);
                    w[i] = *reinterpret_cast<const uint4*>(from + raw_at(lw * 32 + rr, c));
                    f[i] = scale[rr];
                }
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    int rr, c;
                    place(i, rr, c);
                    const int key = lw * 32 + rr;
                    uint8_t* line = to + (c >> 2) * kPanel + key * 128;
                    *reinterpret_cast<uint4*>(line + ((((c & 3) * 2) ^ (key & 7)) * 16)) =
                        make_uint4(mul_half2(e4m3x2_to_f16x2(w[i].x), f[i]), mul_half2(e4m3x2_hi_to_f16x2(w[i].x), f[i]),
                                   mul_half2(e4m3x2_to_f16x2(w[i].y), f[i]), mul_half2(e4m3x2_hi_to_f16x2(w[i].y), f[i]));
                    *reinterpret_cast<uint4*>(line + ((((c & 3) * 2 + 1) ^ (key & 7)) * 16)) =
                        make_uint4(mul_half2(e4m3x2_to_f16x2(w[i].z), f[i]), mul_half2(e4m3x2_hi_to_f16x2(w[i].z), f[i]),
                                   mul_half2(e4m3x2_to_f16x2(w[i].w), f[i]), mul_half2(e4m3x2_hi_to_f16x2(w[i].w), f[i]));
                }
                fence_smem_to_mma();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[slot]);
            }
        } else {
            // Operation n - 1 is handed over once n is on its way, or at once if n has to wait for room.
            auto hand_over = [&](int n) {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                fence_smem_to_mma();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[n % SLOTS]);
            };
            int handed = 0;
            for (int n = 0; ok && n < ops; ++n) {
                const int slot = n % SLOTS;
                const uint32_t parity = ((n / SLOTS) & 1) ^ 1;
                if (!__all_sync(0xffffffffu, mbar_test_wait(&empty[slot], parity))) {
                    for (; handed < n; ++handed) hand_over(handed);
                    ok = mbar_wait_warp(&empty[slot], parity, kBudget, abort);
                    if (!ok) break;
                }
                issue(n, sm + L::kKv + slot * L::kTile);
                commit();
                if (handed < n) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    fence_smem_to_mma();
                    __syncwarp();
                    for (; handed < n; ++handed) {
                        if (lane == 0) mbar_arrive(&full[handed % SLOTS]);
                    }
                }
            }
            for (; ok && handed < ops; ++handed) hand_over(handed);
        }
        if (!ok) *abort = 1;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ---------------------------------------------------------------- softmax
        more_registers<kManyRegs>();
        float c = 1.4426950408889634f / sqrtf(static_cast<float>(D));
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        softmax_sync();
        if constexpr (E4M3) {
            // This thread's row, scaled by a power of two for fp16.
            uint8_t* line = q_tile + r * 128;
            alignas(16) uint32_t w[D / 2];
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                *reinterpret_cast<uint4*>(w + 4 * i) =
                    *reinterpret_cast<const uint4*>(line + (i >> 3) * kPanel + (((i & 7) ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int i = 0; i < D / 2; ++i) {
                big = max3(big, fabsf(a.f16 ? f16_lo(w[i]) : bf16_lo(w[i])),
                           fabsf(a.f16 ? f16_hi(w[i]) : bf16_hi(w[i])));
            }
            int e = 0;
            if (big > 0.0f && big < INFINITY) {
                e = min(13 + 127 - static_cast<int>(__float_as_uint(big) >> 23), 126);
            }
            // Kept a normal number: a masked score is -infinity times it.
            c = fminf(fmaxf(c * pow2(-e) * (exp_of_byte(static_cast<uint32_t>(top_k)) * pow2(-kLift)), 1e-37f), 1e37f);
            if constexpr (!PAIR) softmax_sync();  // both streams have read the row
            if (PAIR || s == 0) {
                const float f = pow2(e);
#pragma unroll
                for (int i = 0; i < D / 2; ++i) {
                    w[i] = pack2_out((a.f16 ? f16_lo(w[i]) : bf16_lo(w[i])) * f,
                                     (a.f16 ? f16_hi(w[i]) : bf16_hi(w[i])) * f, 1);
                }
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    *reinterpret_cast<uint4*>(line + (i >> 3) * kPanel + (((i & 7) ^ (r & 7)) * 16)) =
                        *reinterpret_cast<const uint4*>(w + 4 * i);
                }
            }
        }
        if (PAIR || s == 0) {
            fence_smem_to_mma();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + s * 128, o_at = tmem + lanes + 256 + s * 128;
        float m = -INFINITY, neg = kShift;
        float2 l4[4] = {};
        const int steps = steps_of(s);
        bool ok = true;
        for (int i = 0; i < steps; ++i) {
            const int j = PAIR ? i : 2 * i + s;
            if (!mbar_wait_warp(&s_full[s], i & 1, kBudget, abort)) {
                ok = false;
                break;
            }
            tc_fence_after();
            float x[kKeyTile];
            tmem_ld64(s_at, x);
            tmem_ld64(s_at + 64, x + 64);
            if (mask[j] != 0xff || (tile0 + j + 1) * kKeyTile > a.prefix_len) {
                // Keys that are not there: their page's bit, their place before the end.
                const unsigned pages = mask[j];
                const int left = a.prefix_len - (tile0 + j) * kKeyTile;
#pragma unroll
                for (int k = 0; k < kKeyTile; ++k) {
                    if (!(pages >> (k / kPageTokens) & 1) || k >= left) x[k] = -INFINITY;
                }
            }
            float top4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int k = 4; k < kKeyTile; k += 8) {
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    if (k + z + 4 < kKeyTile) top4[z] = max3_nan(top4[z], x[k + z], x[k + z + 4]);
                    else top4[z] = max_nan(top4[z], x[k + z]);
                }
            }
            const float top = max_nan(max_nan(top4[0], top4[1]), max_nan(top4[2], top4[3])) * c;
            if (__any_sync(0xffffffffu, !(top <= m + kGrow))) {
                const float m_new = max_nan(m, top);
                const float f = m_new == m ? 1.0f : ex2(m - m_new);
                m = m_new;
                // A row that has seen NaN or +infinity stays NaN.
                neg = m < INFINITY ? kShift - (m == -INFINITY ? 0.0f : m) : __int_as_float(0x7fc00000);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    l4[z].x *= f;
                    l4[z].y *= f;
                }
                if (i > 0) {  // the products before this tile's scores are done: O is still
#pragma unroll 1
                    for (int k = 0; k < D / 32; ++k) {
                        float y[32];
                        uint32_t z[32];
                        tmem_ld32(o_at + k * 32, y);
#pragma unroll
                        for (int e = 0; e < 32; ++e) z[e] = __float_as_uint(y[e] * f);
                        tmem_st32(o_at + k * 32, z);
                    }
                }
            }
            const float2 c2 = make_float2(c, c), n2 = make_float2(neg, neg);
            // Half the keys at a time: the product over the first half starts while the second is at work.
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t y[32];
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    float2 p = ffma2(make_float2(x[half * 64 + k], x[half * 64 + k + 1]), c2, n2);
                    p.x = ex2(p.x);
                    p.y = ex2(p.y);
                    x[half * 64 + k] = p.x;
                    x[half * 64 + k + 1] = p.y;
                    y[k / 2] = E4M3 ? pack2_out(p.x, p.y, 1) : weights_hi(p.x, p.y);
                }
                tmem_st32(s_at + half * 32, y);
                if constexpr (!E4M3) {
                    uint32_t lo[32];
#pragma unroll
                    for (int k = 0; k < 64; k += 2) {
                        lo[k / 2] = weights_lo(x[half * 64 + k], x[half * 64 + k + 1], y[k / 2]);
                    }
                    tmem_st32(s_at + 64 + half * 32, lo);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * s + half]);
            }
            // The sum of the weights, while the products run.
#pragma unroll
            for (int k = 0; k < kKeyTile; k += 2) l4[(k >> 1) & 3] = fadd2(l4[(k >> 1) & 3], make_float2(x[k], x[k + 1]));
        }
        // All products are done, of both streams: the operands' room takes the sums, so that they leave as
        // whole rows (16 KB a warp for D = 128; the 16-byte pieces swizzled by their row).
        for (int z = 0; z < 2; ++z) {
            if (ok && steps_of(z) > 0) ok = mbar_wait_warp(&o_full[z], 0, kBudget, abort);
        }
        if (!ok) *abort = 1;
        tc_fence_after();
        float l = ((l4[0].x + l4[0].y) + (l4[1].x + l4[1].y)) + ((l4[2].x + l4[2].y) + (l4[3].x + l4[3].y));
        float f = E4M3 ? exp_of_byte(static_cast<uint32_t>(top_v)) * pow2(-kLift) : 1.0f;
        if constexpr (!PAIR) {
            // Both streams' rows relative to the larger of their maxima.
            float2* ml_s = reinterpret_cast<float2*>(sm + L::kQ);
            ml_s[s * kRowTile + r] = make_float2(m, l);
            softmax_sync();
            const float2 other = ml_s[(s ^ 1) * kRowTile + r];
            const float both = fmaxf(m, other.x);
            const float mine = m == both ? 1.0f : ex2(m - both), theirs = other.x == both ? 1.0f : ex2(other.x - both);
            l = l * mine + other.y * theirs;
            f *= mine;
            m = both;
        }
        constexpr int PIECES = D / 4;  // 16-byte pieces of a row of sums
        float4* mine_s = reinterpret_cast<float4*>(sm + L::kKv) + warp * 32 * PIECES;
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
            float y[32];
            if (ok && steps > 0) {
                tmem_ld32(o_at + k * 32, y);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) y[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                mine_s[lane * PIECES + ((k * 8 + e) ^ (lane & (PIECES - 1)))] =
                    make_float4(y[4 * e] * f, y[4 * e + 1] * f, y[4 * e + 2] * f, y[4 * e + 3] * f);
            }
        }
        tc_fence_before();
        if (live && (PAIR || s == 0)) {
            const float bad = __int_as_float(0x7fc00000);
            a.prefix_ml[part + row] = ok ? make_float2(m, l) : make_float2(bad, bad);
        }
        // The rows this warp writes: its own (PAIR), half of those that both streams have (SOLO).
        constexpr int PER = 32 / PIECES < 1 ? 1 : 32 / PIECES;  // rows at once
        if constexpr (PAIR) __syncwarp();
        else softmax_sync();
        const int first = PAIR ? 0 : s * 16, n_rows = PAIR ? 32 : 16;
        const float4* one = reinterpret_cast<const float4*>(sm + L::kKv) + (PAIR ? warp : warp & 3) * 32 * PIECES;
        const float4* two = one + 4 * 32 * PIECES;
        const int row0 = row_base + (PAIR ? s * kRowTile : 0) + (warp & 3) * 32;
#pragma unroll 4
        for (int i = 0; i < n_rows; i += PER) {
            const int rr = first + i + lane / PIECES, at = rr * PIECES + (lane % PIECES ^ (rr & (PIECES - 1)));
            float4 y = one[at];
            if constexpr (!PAIR) {
                const float4 z = two[at];
                y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
            }
            if (row0 + rr < rows) {
                reinterpret_cast<float4*>(a.prefix_o + (part + row0 + rr) * D)[lane % PIECES] = y;
            }
        }
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
    const dim3 grid(a.prefix_splits, a.n_kv, (rows + tile - 1) / tile);
    constexpr int bytes = Smem<D, E4M3, PAIR>::kBytes;
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

// Parts per row. A CTA's time is about (its key tiles + 3), 3 for its start and end (with 5, 8 or 12 the
// same splits come out at 32768 keys, with 1 others that are 16% slower); the splits make the sum over the
// waves of 148 CTAs least. They do not ask the device, as the workspace's size has to know them too.
//
// The workspace of a batch has to serve every smaller one, but the best splits jump both ways with the number
// of tiles. So they are sought up to most_splits, the best for tiles that could be cut anywhere: for that the
// time is waves(n) * tiles / n + 3 * waves(n), a line over the tiles for each n, flatter and higher for more
// splits, so the least of the lines moves to more splits as tiles grow and never back. (Fewer than 1 choice in
// 100 changes by that, 7% of the time at worst by this count.)
namespace {

struct Cut {
    long long base, tiles, least, most;  // CTAs of one split, key tiles, and splits that are possible
    bool pair;
    Cut(int n_kv, long long rows, int prefix_len) : pair(rows > kRowTile) {
        base = static_cast<long long>(n_kv) * (pair ? (rows + 2 * kRowTile - 1) / (2 * kRowTile) : 1);
        tiles = (static_cast<long long>(prefix_len) + kKeyTile - 1) / kKeyTile;
        least = (tiles + kMaxTiles - 1) / kMaxTiles;
        most = std::max(least, std::min(tiles, 64LL));
    }
    long long waves(long long n) const { return (base * n + 147) / 148; }
    long long most_splits() const {
        long long best = least, best_time = -1;
        for (long long n = least; n <= most; ++n) {
            const long long time = waves(n) * ((pair ? 2 : 1) * tiles + 3 * n);  // n times it
            if (best_time < 0 || time * best <= best_time * n) {
                best = n;
                best_time = time;
            }
        }
        return best;
    }
};

}  // namespace

int prefix_splits(int n_kv, int rows, int prefix_len) {
    if (prefix_len <= 0 || rows <= 0) return 0;
    const Cut cut(n_kv, rows, prefix_len);
    const long long most = cut.most_splits();
    long long best = cut.least, best_time = -1;
    for (long long n = cut.least; n <= most; ++n) {
        const long long each = (cut.tiles + n - 1) / n, time = cut.waves(n) * ((cut.pair ? 2 : 1) * each + 3);
        if (best_time < 0 || time < best_time) {
            best = n;
            best_time = time;
        }
    }
    return static_cast<int>(best);
}

size_t prefix_part_rows(int n_kv, int rows, int prefix_len) {
    if (prefix_len <= 0 || rows <= 0) return 0;
    // The most rows of each number of row tiles: one tile alone, then pairs.
    long long most = std::min(rows, kRowTile) * Cut(n_kv, 1, prefix_len).most_splits();
    for (long long n = 2 * kRowTile; rows > kRowTile; n += 2 * kRowTile) {
        most = std::max(most, std::min<long long>(rows, n) * Cut(n_kv, n, prefix_len).most_splits());
        if (n >= rows) break;
    }
    return static_cast<size_t>(most);
}

void launch_prefix_attention(const PagedArgs& a, int head_dim, bool e4m3, cudaStream_t s) {
    if (head_dim == 64) launch<64>(a, e4m3, s);
    else launch<128>(a, e4m3, s);
}

}  // namespace q3
