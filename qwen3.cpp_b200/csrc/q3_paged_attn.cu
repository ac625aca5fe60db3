// q3_paged_attn / q3_prefix_attn: attention of a ragged batch's newest rows over a paged KV pool,
// with or without a prefix that every sequence shares.
//
// own_pages_kernel computes the part over each sequence's own pages (and over a short prefix, whose pages
// then stand in front of them), join_kernel joins parts.
//
// Work: a strip is the pages of one (sequence, KV head, group of 8 * NT rows). Where tables are short
// each strip is one block's, which finishes its rows. Else a strip's units are its pages and kSetup more
// in front, for what a strip costs before and after its pages. The units of all sequences form one line,
// cut into equal runs, one a block, so a ragged batch loads every block alike and a long sequence spreads
// over many. Each block finds its run from the lengths on the device (a scan over the sequences), so a
// captured graph follows them. A strip whose pages lie inside one run is finished there; one that is cut
// leaves a part per block, at most two a block, and join_kernel adds them by their softmax statistics.
//
// A block's warps take a page each in turn. A page is 16 keys, one m16n8k16 operand tile:
//   S^T[16 keys x 8 rows] = K . Q^T      K's rows are the A operand as they lie in memory
//   O^T[d x 8 rows]      += V^T . P^T    two keys' V values of one d are a register of A
// The order of the head's dimensions inside an operand is free as long as both sides agree, so a lane
// takes 16 contiguous bytes and they are its operand registers (bf16) or become them by a conversion
// (e4m3 -> fp16, exact); V pairs need one byte permutation. The scores come out transposed for the
// second product; movmatrix turns the rounded weights.
//
// Each warp has its own ring of two pages in shared memory, filled by cp.async a page ahead (three pages:
// 64 sequences of 128 to 4096 tokens 56.3 us instead of 53.5, 16 of 5 rows and 100 to 5000 tokens 36.8
// instead of 37.1). 16-byte piece c of row r lies at piece c ^ (r % 8), which leaves the operand reads
// without bank conflicts.
//
// A row's running maximum moves only when a weight passes it by more than 2^4 (one vote a page instead of two
// times three shuffles). In an e4m3 pool the weight that meets V is p times the power of two of the V row,
// which fp16 has to hold: the maximum is that of these products over the keys that the row sees. What fp16 cuts
// off is then 2^-33 of the row's largest weighted V row, whatever rows hold that have no weight or that later
// rows alone see. The sum of p, in fp32, has room for p of 2^64 before its own reference moves. The largest
// weight is 2^kShift and so not rounded, which counts where one key dominates (references rounded up to whole
// powers of two, or left alone up to 2^7, came to 2 and 1.1 times the error of fp16 results, 1% faster at most).
//
// Rounding: e4m3 -> fp16 is exact; a query row is scaled by a power of two so that its largest value
// is in [2^13, 2^14): bf16 and fp16 values are then fp16 values down to 2^-38 of the row's largest.
// Weights, with V's power of two, are rounded to fp16 (2^-11), for a bf16 pool to a bf16 pair hi + lo (2^-16).
// Sums are fp32.
//
// Bound by HBM: 2 * (D + 1) bytes a key and KV head (e4m3). 64 sequences of 128 to 4096 tokens, 8 KV heads
// of 128: 279 MB in 52.9 us, 5.3 TB/s with the start, the last blocks and the join, about 6 TB/s between
// them; a page costs about 405 warp instructions, which keeps the integer pipe half busy. Past 16 rows a KV head
// every page is read (from L2) and multiplied once per 16 rows, and instructions bound: 8 query heads to a KV head,
// 64 sequences as above, 1, 2, 5 and 16 rows each take 55.6, 74.6, 175 and 501 us.
#include <algorithm>
#include <climits>

#include "q3_paged_attn.cuh"

namespace q3 {

namespace {

constexpr int kWarps = 4;                // of a block on the line, and of the join
constexpr int kThreads = kWarps * 32;
constexpr int kStripWarps = 8;           // of a strip's block where there are few strips
// log2 of the largest p (bf16 pool) or p times V's power of two (e4m3), and for e4m3 of the largest p, that leave
// their references where they are.
constexpr float kTop = kShift + 4.0f, kTopE4m3 = 64.0f;
constexpr float kUnseen = 1e38f;  // reference of a row that has seen no key: any score then passes the top

// Tables of up to so many pages take a block a strip: 1 sequence of 512 tokens 7.4 us against 8.4 with
// the line, whose scan and join cost about 4 us. The table's width decides, as the lengths are on the device.
constexpr int kStripPages = 64;

// A prefix this short (pages, the sequence's own among them) for this little work (strips x prefix pages)
// is read by each strip in front of its own pages, from L2 after the first: one launch instead of two.
// (30 sequences of 2 rows, 4 KV heads, 300 shared tokens: 7.8 us against 15.1; 100 of 1 row, 8 heads, 160
// tokens: 16.9 against 22.1; 1000 tokens, past the limit, would take 40 against 24.)
constexpr int kInlinePages = 96, kInlineWork = 16384;

// How the blocks share the work: a run of the line each, or a strip each with kWarps or kStripWarps warps.
enum Mode { kLine, kStrip, kWideStrip };

// Warps of a block, pages of a warp's ring, and blocks a multiprocessor (registers and rings together).
// Heads of 64 leave room for one more: strips of 200 x 4 rows and 100 tokens 28.4 -> 25.8 us, a bf16 pool's
// line of 40 x 4 rows and 100 to 4000 tokens 26.0 -> 24.6; an e4m3 pool's line is slower for it (64 x 128 to
// 4096: 40.4 against 36.0).
template <int D, bool E4M3, int NT, Mode MODE>
struct Shape {
    static constexpr int kWarps = MODE == kWideStrip ? kStripWarps : q3::kWarps;
    static constexpr int kStages = 2;
    static constexpr int kBlocks = MODE == kWideStrip ? (NT == 1 && E4M3 ? 2 : 1)
                                                      : (NT == 1 ? (E4M3 ? 4 : 3) : (E4M3 ? 3 : 2)) +
                                                            (D == 64 && (MODE == kStrip || !E4M3));
};

__device__ __forceinline__ void copy_16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_16(uint32_t from, uint32_t* r) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(from) : "memory");
}
__device__ __forceinline__ void lds_8(uint32_t from, uint32_t* r) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(from) : "memory");
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t from) {
    uint16_t r;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(from) : "memory");
    return r;
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (F16) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// The same onto zeros.
template <bool F16>
__device__ __forceinline__ void mma16816_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (F16) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Whether a packed word of pool values holds an infinity or NaN.
template <bool E4M3>
__device__ __forceinline__ bool odd_word(uint32_t x) {
    return E4M3 ? (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0
                : (((x & 0x7fff7fffu) + 0x00800080u) & 0x80008000u) != 0;
}

// Piece j (of PIECES / 4) that lane t of its row's four takes of a K row, and of a Q row: neighbours, so
// that two rows' reads fall into different banks.
template <int PIECES>
__device__ __forceinline__ int k_piece(int t, int j) {
    return PIECES == 4 ? t : (j >> 1) * 8 + 2 * t + (j & 1);
}

// The A operand of O^T += V^T P^T for m-tile i: a0, a1 from the keys 2t, 2t + 1, a2, a3 from 2t + 8,
// 2t + 9 (t = lane % 4), for the lane's values 2i and 2i + 1 of each.
template <bool E4M3, int VW>
__device__ __forceinline__ void v_operand(const uint32_t (&vr)[4][VW], int i, uint32_t (&f)[4]) {
    if constexpr (E4M3) {
        const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
        const uint32_t p0 = __byte_perm(vr[0][i >> 1], vr[1][i >> 1], sel);
        const uint32_t p1 = __byte_perm(vr[2][i >> 1], vr[3][i >> 1], sel);
        f[0] = e4m3x2_to_f16x2(p0);
        f[1] = e4m3x2_hi_to_f16x2(p0);
        f[2] = e4m3x2_to_f16x2(p1);
        f[3] = e4m3x2_hi_to_f16x2(p1);
    } else {
        f[0] = __byte_perm(vr[0][i], vr[1][i], 0x5410u);
        f[1] = __byte_perm(vr[0][i], vr[1][i], 0x7632u);
        f[2] = __byte_perm(vr[2][i], vr[3][i], 0x5410u);
        f[3] = __byte_perm(vr[2][i], vr[3][i], 0x7632u);
    }
}

// Threads' sums of units, one after the other: the sums before this thread and of all.
__device__ __forceinline__ void block_scan(long long mine, long long* warp_sums, long long& before,
                                           long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    before = x - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
}

// Units of a strip; one without pages has one all the same, so that a block sees to its rows.
__device__ __forceinline__ int strip_units(int pages) { return max(pages, 1) + kSetup; }

template <int NT>
__device__ __forceinline__ int row_groups(const SeqShape& s, int group) {
    return (s.rows * group + 8 * NT - 1) / (8 * NT);
}

// Joins one row's n parts and writes its head, by one warp: a lane looks up a part's weight and place
// (part_of(i, ml, o)), then all lanes add the part's sums, several parts on their way at once. The
// order is the parts', whoever joins them.
// It starts from a part that the warp already has: (top, its sum in lane 0 and 0 elsewhere, y).
template <int D, typename PartOf>
__device__ __forceinline__ void join_row(float top, float sum, float (&y)[D / 32], int n, PartOf part_of,
                                         uint16_t* out, int f16) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    for (int i0 = 0; i0 < n; i0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.0f);
        const float* o = nullptr;
        if (i0 + lane < n) {
            const float2* p;
            part_of(i0 + lane, p, o);
            ml = __ldcg(p);
        }
        const float top_new = fmaxf(top, warp_max(ml.x));
        const float back = top_new == top ? 1.0f : ex2(top - top_new);
        const float f = ml.x == top_new ? 1.0f : ex2(ml.x - top_new);
        top = top_new;
        sum = fmaf(ml.y, f, sum * back);
#pragma unroll
        for (int d = 0; d < V; ++d) y[d] *= back;
        const int here = min(32, n - i0);
#pragma unroll 8
        for (int x = 0; x < here; ++x) {
            const float* ox = reinterpret_cast<const float*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o), x));
            const float fx = __shfl_sync(0xffffffffu, f, x);
            float z[V];
            if constexpr (V == 4) *reinterpret_cast<float4*>(z) = __ldcg(reinterpret_cast<const float4*>(ox + lane * V));
            else *reinterpret_cast<float2*>(z) = __ldcg(reinterpret_cast<const float2*>(ox + lane * V));
#pragma unroll
            for (int d = 0; d < V; ++d) y[d] = fmaf(z[d], fx, y[d]);
        }
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing is zeros
    uint32_t z[V / 2];
#pragma unroll
    for (int d = 0; d < V; d += 2) z[d / 2] = pack2_out(y[d] * inv, y[d + 1] * inv, f16);
    if constexpr (V == 4) *reinterpret_cast<uint2*>(out + lane * V) = make_uint2(z[0], z[1]);
    else *reinterpret_cast<uint32_t*>(out + lane * V) = z[0];
}

template <int NT>
__device__ __forceinline__ long long seq_units(const PagedArgs& a, const SeqShape& s) {
    return static_cast<long long>(a.n_kv) * row_groups<NT>(s, a.group) * strip_units(seq_pages(s));
}

// Units of one block's run.
__device__ __forceinline__ long long run_length(long long total, unsigned blocks) {
    return max(static_cast<long long>(kMinUnits), (total + blocks - 1) / static_cast<long long>(blocks));
}

template <int D, bool E4M3, int NT, Mode MODE>
struct OwnSmem {
    static constexpr int kRow = E4M3 ? D : 2 * D;                  // bytes of a pool row
    static constexpr int kPage = 2 * kPageTokens * kRow + (E4M3 ? 2 * kPageTokens : 0);  // K, V, bytes
    static constexpr int kRing = Shape<D, E4M3, NT, MODE>::kWarps * Shape<D, E4M3, NT, MODE>::kStages * kPage;
    static constexpr int kSums = Shape<D, E4M3, NT, MODE>::kWarps * 8 * NT * D * 4;          // after a run of pages, in its place
    static constexpr int kBytes = kRing > kSums ? kRing : kSums;
};

// kLine: the block takes its run of the line of units. Else it takes one strip and finishes its rows,
// the prefix's parts among them.
template <int D, bool E4M3, int NT, Mode MODE>
__global__ void __launch_bounds__(Shape<D, E4M3, NT, MODE>::kWarps * 32, Shape<D, E4M3, NT, MODE>::kBlocks)
    own_pages_kernel(const PagedArgs a) {
    constexpr int MT = D / 16;                    // m-tiles of O^T, k-steps of S^T
    constexpr int KW = E4M3 ? D / 16 : D / 8;     // words a lane holds of one K row
    constexpr int VW = E4M3 ? D / 32 : D / 16;    // and of one V row
    using L = OwnSmem<D, E4M3, NT, MODE>;
    constexpr int W = Shape<D, E4M3, NT, MODE>::kWarps;
    constexpr bool LINE = MODE == kLine;
    constexpr int ROW = L::kRow, PIECES = ROW / 16, STAGES = Shape<D, E4M3, NT, MODE>::kStages;
    constexpr int ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t ring_s[];
    float (*o_s)[ROWS][D] = reinterpret_cast<float (*)[ROWS][D]>(ring_s);
    __shared__ float m_s[W][ROWS], l_s[W][ROWS];
    __shared__ long long scan_s[W];
    __shared__ long long first_s;
    __shared__ int seq_s;

    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring_s)) + warp * STAGES * L::kPage;
    const float scale = 1.4426950408889634f / sqrtf(static_cast<float>(D));
    long long pos = 0, end = 1, seq_first = 0;
    int b, h, rg, ids = -1;
    if constexpr (LINE) {
        // This block's run of units.
        const int per_thread = (a.n_seqs + W * 32 - 1) / (W * 32);
        const int b0 = min(tid * per_thread, a.n_seqs), b1 = min(b0 + per_thread, a.n_seqs);
        auto units = [&](int i) { return seq_units<NT>(a, seq_shape(a, i)); };
        long long mine = 0, before, total;
        for (int i = b0; i < b1; ++i) mine += units(i);
        block_scan(mine, scan_s, before, total);
        const long long per = run_length(total, gridDim.x);
        pos = per * blockIdx.x;
        end = min(total, pos + per);
        if (pos >= end) {
            pdl_wait();
            return;
        }
        if (before <= pos && pos < before + mine) {
            long long x = before;
            int i = b0;
            for (long long u; x + (u = units(i)) <= pos; ++i) x += u;
            seq_s = i;
            first_s = x;
        }
        __syncthreads();
        seq_first = first_s;
        b = seq_s;
    } else {
        const unsigned most = (a.max_q * a.group + ROWS - 1) / ROWS;
        rg = static_cast<int>(blockIdx.x % most);
        h = static_cast<int>(blockIdx.x / most % a.n_kv);
        b = static_cast<int>(blockIdx.x / most / a.n_kv);
        // The first pages' numbers are on their way with the lengths.
        const int p = warp + lane * W - a.inline_pages;
        if (p < 0) ids = a.prefix_table[p + a.inline_pages];
        else if (p < a.table_stride) ids = a.table[static_cast<size_t>(b) * a.table_stride + p];
    }
    while (pos < end) {
        const SeqShape s = seq_shape(a, b);
        const int pages = seq_pages(s), groups = row_groups<NT>(s, a.group);
        int p0 = 0, p1 = pages;
        const int before = LINE ? 0 : a.inline_pages;  // of the prefix, in front of the strip's own
        if constexpr (LINE) {
            const int each = strip_units(pages);
            const long long all = static_cast<long long>(a.n_kv) * groups * each;
            if (pos >= seq_first + all) {
                seq_first += all;
                ++b;
                continue;
            }
            const long long strip = (pos - seq_first) / each;  // (head, row group)
            const long long strip_first = seq_first + strip * each;
            const long long u1 = min(strip_first + each, end);
            // This block's pages of it: all of them, or the run's beginning or end cuts them.
            p0 = static_cast<int>(max(0LL, pos - strip_first - kSetup));
            p1 = min(pages, static_cast<int>(u1 - strip_first) - kSetup);
            pos = u1;
            if (u1 - strip_first <= kSetup) continue;  // the run ends in front of the strip's first page
            h = static_cast<int>(strip / groups);
            rg = static_cast<int>(strip % groups);
        } else {
            pos = end;
            if (rg >= groups) break;
            p1 += before;
        }
        const int r_base = rg * ROWS;
        const int n_rows = min(ROWS, s.rows * a.group - r_base);

        // This warp's pages, the first of them on their way.
        const int32_t* table = a.table + static_cast<size_t>(b) * a.table_stride;
        const int steps = p1 - p0 > warp ? (p1 - p0 - warp + W - 1) / W : 0;
        uint32_t fill = ring, page_s = ring;  // the ring's next page to fill, to use
        unsigned good = 0;  // of the last 32 steps looked up: whether the page is in the pool
        auto start_page = [&](int it) {  // in order: 0, 1, 2, ...
            if ((it & 31) == 0 && (LINE || it > 0)) {
                const int p = p0 + warp + (it + lane) * W;
                ids = p >= p1 ? -1 : p < before ? a.prefix_table[p] : table[p - before];
            }
            const int page = __shfl_sync(0xffffffffu, ids, it & 31);
            const bool in = page >= 0 && page < a.n_pages;
            good = good << 1 | in;
            // A page that is not there is page 0 in its place, whose keys are masked.
            const size_t row = (static_cast<size_t>(in ? page : 0) * a.n_kv + h) * kPageTokens;
            const uint32_t to = fill;
            fill = fill == ring + (STAGES - 1) * L::kPage ? ring : fill + L::kPage;
            const uint8_t* kp = static_cast<const uint8_t*>(a.k) + row * ROW;
            const uint8_t* vp = static_cast<const uint8_t*>(a.v) + row * ROW;
#pragma unroll
            for (int i = 0; i < kPageTokens * PIECES / 32; ++i) {
                const int x = i * 32 + lane, r = x / PIECES, c = x % PIECES;
                const uint32_t at = r * ROW + ((c ^ (r & (PIECES < 8 ? PIECES - 1 : 7))) * 16);
                copy_16(to + at, kp + x * 16);
                copy_16(to + kPageTokens * ROW + at, vp + x * 16);
            }
            if (E4M3 && lane < 8) {
                copy_4(to + 2 * kPageTokens * ROW + lane * 4, a.exps + row * 2 + lane * 4);
            }
        };
#pragma unroll
        for (int it = 0; it < STAGES - 1; ++it) {
            if (it < steps) start_page(it);
            copy_commit();
        }

        // Q as the B operand: lane (g, t) holds row g's values in the order of K's.
        uint32_t qw[NT][D / 8];
        float c_col[E4M3 ? NT : 1][2];  // score factor of the columns 2t, 2t + 1 (a bf16 pool has one for all)
        c_col[0][0] = scale;
        int seen[NT][2];  // keys that their rows see, none for a row past the last
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = r_base + n * 8 + g;
            const bool live = n * 8 + g < n_rows;
            const int token = token_of(a, r);
            const uint16_t* qp = static_cast<const uint16_t*>(a.q) +
                                 (live ? (s.row0 + token) * a.q_stride + (h * a.group + r - token * a.group) * D : 0);
            constexpr int CH = E4M3 ? 16 : 8;  // values of a 16-byte piece
#pragma unroll
            for (int j = 0; j < PIECES / 4; ++j) {
#pragma unroll
                for (int i = 0; i < CH / 8; ++i) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (live) x = *reinterpret_cast<const uint4*>(qp + k_piece<PIECES>(t, j) * CH + 8 * i);
                    uint32_t* w = &qw[n][(j * (CH / 8) + i) * 4];
                    w[0] = x.x;
                    w[1] = x.y;
                    w[2] = x.z;
                    w[3] = x.w;
                }
            }
            if constexpr (E4M3) {
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const float lo = a.f16 ? f16_lo(qw[n][i]) : bf16_lo(qw[n][i]);
                    const float hi = a.f16 ? f16_hi(qw[n][i]) : bf16_hi(qw[n][i]);
                    big = fmaxf(big, fmaxf(fabsf(lo), fabsf(hi)));
                }
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                int e = 0;
                if (big > 0.0f && big < INFINITY) {
                    e = min(13 + 127 - static_cast<int>(__float_as_uint(big) >> 23), 126);
                }
                const float f = pow2(e);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const float lo = a.f16 ? f16_lo(qw[n][i]) : bf16_lo(qw[n][i]);
                    const float hi = a.f16 ? f16_hi(qw[n][i]) : bf16_hi(qw[n][i]);
                    qw[n][i] = pack2_out(lo * f, hi * f, 1);
                }
                const float c = scale * pow2(-e);
#pragma unroll
                for (int x = 0; x < 2; ++x) c_col[n][x] = __shfl_sync(0xffffffffu, c, (2 * t + x) * 4);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int rr = n * 8 + 2 * t + x;
                seen[n][x] = rr < n_rows ? s.len - s.rows + token_of(a, r_base + rr) + 1 : 0;
            }
        }
        const int tail_key = s.len - s.rows + token_of(a, r_base) + 1;  // seen by every row below it

        // l = sum 2^(score + neg), o = sum 2^(score + neg) * v (bf16 pool), or of 2^(score + log2 of V's power +
        // neg_v) * V's codes (e4m3). The references neg and neg_v are kShift - the maximum.
        float neg[NT][2], neg_v[NT][2], l[NT][2], o[NT][MT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                neg[n][x] = kUnseen;
                if constexpr (E4M3) neg_v[n][x] = kUnseen;
                l[n][x] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        }

        for (int it = 0; it < steps; ++it) {
            const int p_here = p0 + warp + it * W;
            const bool shared = !LINE && p_here < before;  // a page of the prefix: all rows see all its keys
            const int key0 = (shared ? p_here : p_here - before) * kPageTokens;
            copy_wait<STAGES - 2>();
            __syncwarp();  // every lane's copies of this page are in, and its reads of the one before done
            // `good` grows a bit a page looked up: this page's is (pages looked up since) from its end.
            const bool there = good >> (min(it + STAGES - 2, steps - 1) - it) & 1;
            if (it + STAGES - 1 < steps) start_page(it + STAGES - 1);
            copy_commit();
            constexpr int SW = PIECES < 8 ? PIECES - 1 : 7;
            // All of K's pieces at once.
            uint32_t kr[2][KW], ex[2] = {0, 0};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int j = 0; j < PIECES / 4; ++j) {
                    lds_16(page_s + (g + 8 * x) * ROW + ((k_piece<PIECES>(t, j) ^ (g & SW)) * 16), &kr[x][4 * j]);
                }
            }
            if constexpr (E4M3) {
                ex[0] = lds_u16(page_s + 2 * kPageTokens * ROW + g * 2);
                ex[1] = lds_u16(page_s + 2 * kPageTokens * ROW + g * 2 + 16);
            }
            float sc[NT][4];
#pragma unroll
            for (int k = 0; k < MT; ++k) {
                uint32_t f[4];
                if constexpr (E4M3) {
                    f[0] = e4m3x2_to_f16x2(kr[0][k]);
                    f[1] = e4m3x2_to_f16x2(kr[1][k]);
                    f[2] = e4m3x2_hi_to_f16x2(kr[0][k]);
                    f[3] = e4m3x2_hi_to_f16x2(kr[1][k]);
                } else {
                    f[0] = kr[0][2 * k];
                    f[1] = kr[1][2 * k];
                    f[2] = kr[0][2 * k + 1];
                    f[3] = kr[1][2 * k + 1];
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (k == 0) mma16816_new<E4M3>(sc[n], f[0], f[1], f[2], f[3], qw[n][0], qw[n][1]);
                    else mma16816<E4M3>(sc[n], f[0], f[1], f[2], f[3], qw[n][2 * k], qw[n][2 * k + 1]);
                }
            }
            const bool tail = !there || key0 + kPageTokens > (shared ? a.prefix_len : tail_key);
            const int limit = there ? (shared ? a.prefix_len : s.len) - key0 : 0;  // this page's keys that exist
            const float k_factor[2] = {exp_of_byte(ex[0] & 0xffu), exp_of_byte(ex[1] & 0xffu)};
            float p[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[n][i] = sc[n][i] * (E4M3 ? c_col[n][i & 1] : c_col[0][0]);
                    if constexpr (E4M3) p[n][i] *= k_factor[i >> 1];
                }
            }
            if (tail) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = g + 8 * (i >> 1);
                        if (k >= limit || (!shared && key0 + k >= seen[n][i & 1])) p[n][i] = -INFINITY;
                    }
                }
            }
            // log2 of V's powers of two. (A key that is not there has a score of -infinity, whatever its byte.)
            float v_log[2] = {0.0f, 0.0f};
            if constexpr (E4M3) {
#pragma unroll
                for (int x = 0; x < 2; ++x) v_log[x] = __uint_as_float(0x4b000000u | ex[x] >> 8) - (8388608.0f + 127.0f);
            }
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    grow |= p[n][i] + neg[n][i & 1] > (E4M3 ? kTopE4m3 : kTop);
                    if constexpr (E4M3) grow |= p[n][i] + (v_log[i >> 1] + neg_v[n][i & 1]) > kTop;
                }
            }
            if (__any_sync(0xffffffffu, grow)) {
                // `at` down to kShift - the page's largest, in each column.
                auto move = [](float (&at)[NT][2], float (&largest)[NT][2], float (&factor)[NT][2]) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                largest[n][x] = fmaxf(largest[n][x], __shfl_xor_sync(0xffffffffu, largest[n][x], o));
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float to = fminf(at[n][x], kShift - largest[n][x]);
                            factor[n][x] = ex2(to - at[n][x]);
                            at[n][x] = to;
                        }
                    }
                };
                float largest[NT][2], f[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) largest[n][x] = fmaxf(p[n][x] + v_log[0], p[n][x + 2] + v_log[1]);
                }
                move(E4M3 ? neg_v : neg, largest, f);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        o[n][i][0] *= f[n][0];
                        o[n][i][1] *= f[n][1];
                        o[n][i][2] *= f[n][0];
                        o[n][i][3] *= f[n][1];
                    }
                }
                if constexpr (!E4M3) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) l[n][x] *= f[n][x];
                    }
                } else {
                    // A row's first neg goes by neg_v and the page's largest power, which leaves the largest p at
                    // 2^kShift or more; what is too far above gets one of its own.
                    const float v_top = static_cast<float>(__reduce_max_sync(0xffffffffu, max(ex[0] >> 8, ex[1] >> 8))) - 127.0f;
                    grow = false;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (neg[n][x] == kUnseen && neg_v[n][x] != kUnseen) neg[n][x] = neg_v[n][x] + v_top;
                            largest[n][x] = fmaxf(p[n][x], p[n][x + 2]);
                            grow |= largest[n][x] + neg[n][x] > kTopE4m3;
                        }
                    }
                    if (__any_sync(0xffffffffu, grow)) {
                        move(neg, largest, f);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) l[n][x] *= f[n][x];
                        }
                    }
                }
            }
            uint32_t pb[NT][2], pl[NT][2];  // P^T as the B operand (and its low half)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float w[2];  // of key x in the columns 2t, 2t + 1
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float score = p[n][2 * x + i];
                        w[i] = ex2(score + neg[n][i]);
                        l[n][i] += w[i];
                        if constexpr (E4M3) w[i] = ex2(score + (v_log[x] + neg_v[n][i]));
                    }
                    if constexpr (E4M3) {
                        pb[n][x] = transpose8x8(pack2_out(w[0], w[1], 1));
                    } else {
                        const uint32_t hi = weights_hi(w[0], w[1]);
                        pb[n][x] = transpose8x8(hi);
                        pl[n][x] = transpose8x8(weights_lo(w[0], w[1], hi));
                    }
                }
            }
            // O^T += V^T P^T, a 16-byte piece of the four keys at a time.
            constexpr int VP = VW < 4 ? VW : 4;  // words of a piece
            bool odd_any = false;
#pragma unroll
            for (int j = 0; j < VW / VP; ++j) {
                uint32_t vr[4][VP];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = 2 * t + (x & 1) + 8 * (x >> 1);
                    const uint32_t at = page_s + (kPageTokens + r) * ROW;
                    if constexpr (VP == 2) lds_8(at + (((g >> 1) ^ (r & SW)) * 16) + (g & 1) * 8, vr[x]);
                    else lds_16(at + (((j * 8 + g) ^ (r & SW)) * 16), vr[x]);
                }
                if (tail) {
                    // Values of keys that are not there are anything, NaN too: as zeros they add nothing.
                    bool odd = false;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const bool here = 2 * t + (x & 1) + 8 * (x >> 1) < limit;
#pragma unroll
                        for (int w = 0; w < VP; ++w) {
                            vr[x][w] = here ? vr[x][w] : 0u;
                            odd |= odd_word<E4M3>(vr[x][w]);
                        }
                    }
                    odd_any = __any_sync(0xffffffffu, odd);
                }
                constexpr int TILES = MT / (VW / VP);
                if (tail && odd_any) {
                    // An infinity or NaN that some rows see and others do not: token by token, with the keys
                    // that the token does not see as zeros.
                    const int first = r_base / a.group, last = (r_base + n_rows - 1) / a.group;
                    for (int tok = first; tok <= last; ++tok) {
                        const int lim = shared ? limit : there ? s.len - s.rows + tok + 1 - key0 : 0;
                        uint32_t vm[4][VP];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const bool here = 2 * t + (x & 1) + 8 * (x >> 1) < lim;
#pragma unroll
                            for (int w = 0; w < VP; ++w) vm[x][w] = here ? vr[x][w] : 0u;
                        }
#pragma unroll
                        for (int i = 0; i < TILES; ++i) {
                            uint32_t f[4];
                            v_operand<E4M3, VP>(vm, i, f);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma16816<E4M3>(c, f[0], f[1], f[2], f[3], pb[n][0], pb[n][1]);
                                if constexpr (!E4M3) mma16816<false>(c, f[0], f[1], f[2], f[3], pl[n][0], pl[n][1]);
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    if ((r_base + n * 8 + 2 * t + (q & 1)) / a.group == tok) o[n][j * TILES + i][q] += c[q];
                                }
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < TILES; ++i) {
                        uint32_t f[4];
                        v_operand<E4M3, VP>(vr, i, f);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816<E4M3>(o[n][j * TILES + i], f[0], f[1], f[2], f[3], pb[n][0], pb[n][1]);
                            if constexpr (!E4M3) {
                                mma16816<false>(o[n][j * TILES + i], f[0], f[1], f[2], f[3], pl[n][0], pl[n][1]);
                            }
                        }
                    }
                }
            }
            page_s = page_s == ring + (STAGES - 1) * L::kPage ? ring : page_s + L::kPage;
        }

        // Join the warps.
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 4);
                l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 8);
                l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 16);
                if constexpr (E4M3) {
                    // Down to a sum of less than 2^(kShift + 1), so that o in its units stays in range.
                    const int k = max((__float_as_int(l[n][x]) >> 23 & 0xff) - 127 - static_cast<int>(kShift), 0);
                    l[n][x] *= __int_as_float((127 - k) << 23);
                    neg[n][x] -= static_cast<float>(k);
                }
                if (g == 0) {
                    m_s[warp][n * 8 + 2 * t + x] = neg[n][x] == kUnseen ? -INFINITY : kShift - neg[n][x];
                    l_s[warp][n * 8 + 2 * t + x] = l[n][x];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = n * 8 + 2 * t + x;
                float top = m_s[0][r];
#pragma unroll
                for (int w = 1; w < W; ++w) top = fmaxf(top, m_s[w][r]);
                const float mine = m_s[warp][r];
                float f = mine == top ? 1.0f : ex2(mine - top), f_v = 1.0f;
                if constexpr (E4M3) {
                    // From neg_v to neg, in two steps: 2^127 and 2^-127 come up.
                    f_v = ex2(0.5f * (neg[n][x] - neg_v[n][x]));
                    f *= f_v;
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int v0 = 2 * i;  // the lane's values 2i, 2i + 1 are neighbours
                    const int d = E4M3 ? g * (D / 8) + v0 : (v0 / 8) * 64 + g * 8 + v0 % 8;
                    *reinterpret_cast<float2*>(&o_s[warp][r][d]) =
                        make_float2(o[n][i][x] * f * f_v, o[n][i][x + 2] * f * f_v);
                }
            }
        }
        __syncthreads();
        if constexpr (!LINE) {
            // A strip's block has its rows to itself: a warp a row, the prefix's parts behind its own.
            pdl_wait();
            const size_t split = static_cast<size_t>(a.n_kv) * a.prefix_rows;
            for (int r = warp; r < n_rows; r += W) {
                constexpr int V = D / 32;
                float top = m_s[0][r], sum = 0.0f, y[V] = {};
#pragma unroll
                for (int w = 1; w < W; ++w) top = fmaxf(top, m_s[w][r]);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    sum += l_s[w][r] * (m_s[w][r] == top ? 1.0f : ex2(m_s[w][r] - top));
#pragma unroll
                    for (int d = 0; d < V; ++d) y[d] += o_s[w][r][lane * V + d];
                }
                const int rr = r_base + r;
                const size_t row = h * static_cast<size_t>(a.prefix_rows) + static_cast<size_t>(s.row0) * a.group + rr;
                join_row<D>(
                    top, lane == 0 ? sum : 0.0f, y, a.prefix_splits,
                    [&](int i, const float2*& ml, const float*& o) {
                        ml = a.prefix_ml + i * split + row;
                        o = a.prefix_o + (i * split + row) * D;
                    },
                    static_cast<uint16_t*>(a.out) + (s.row0 + token_of(a, rr)) * a.out_stride +
                        (h * a.group + rr - token_of(a, rr) * a.group) * D,
                    a.f16);
            }
            break;
        }
        const bool whole = p0 == 0 && p1 == pages;
        const int part = p0 > 0 ? 0 : 1;
        for (int at = tid; at < n_rows * (D / 4); at += W * 32) {
            const int r = at / (D / 4), d = at % (D / 4) * 4;
            float top = m_s[0][r];
#pragma unroll
            for (int w = 1; w < W; ++w) top = fmaxf(top, m_s[w][r]);
            float sum = 0.0f;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                sum += l_s[w][r] * (m_s[w][r] == top ? 1.0f : ex2(m_s[w][r] - top));
                const float4 z = *reinterpret_cast<const float4*>(&o_s[w][r][d]);
                y.x += z.x;
                y.y += z.y;
                y.z += z.z;
                y.w += z.w;
            }
            if (whole && a.prefix_len == 0) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing is zeros
                const int rr = r_base + r;
                const int token = token_of(a, rr);
                uint16_t* out = static_cast<uint16_t*>(a.out) + (s.row0 + token) * a.out_stride +
                                (h * a.group + rr - token * a.group) * D + d;
                *reinterpret_cast<uint2*>(out) = make_uint2(pack2_out(y.x * inv, y.y * inv, a.f16),
                                                            pack2_out(y.z * inv, y.w * inv, a.f16));
            } else if (whole) {
                const size_t row = h * static_cast<size_t>(a.prefix_rows) +
                                   static_cast<size_t>(s.row0) * a.group + r_base + r;
                *reinterpret_cast<float4*>(a.whole_o + row * D + d) = y;
                if (d == 0) a.whole_ml[row] = make_float2(top, sum);
            } else {
                const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + part;
                *reinterpret_cast<float4*>(a.own_o + (slot * ROWS + r) * D + d) = y;
                if (d == 0) a.own_ml[slot * ROWS + r] = make_float2(top, sum);
            }
        }
        __syncthreads();
    }
    // On the line this grid may have started beside the prefix's, which it does not read; join_kernel waits
    // for this one alone, so this one ends after that.
    pdl_wait();
}

// Joins the rows that have several parts: those of the prefix, and of the sequence's own pages one
// where a block did the whole strip and one a block where they cut it. A warp a row. It finds the
// blocks' runs from the lengths again, while own_pages_kernel is still at work.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) join_kernel(const PagedArgs a, const unsigned blocks) {
    constexpr int ROWS = 8 * NT;
    const int most = a.max_q * a.group, lane = threadIdx.x & 31;
    const long long w = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int r = static_cast<int>(w % most), h = static_cast<int>(w / most % a.n_kv);
    const long long b = w / most / a.n_kv;
    // Every block waits, also one with nothing to do: what comes after this grid comes after both.
    if (b >= a.n_seqs) {
        pdl_wait();
        return;
    }
    const SeqShape s = seq_shape(a, static_cast<int>(b));
    long long before = 0, total = 0;
    for (int i = lane; i < a.n_seqs; i += 32) {
        const long long u = seq_units<NT>(a, seq_shape(a, i));
        total += u;
        if (i < b) before += u;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    const int each = strip_units(seq_pages(s)), groups = row_groups<NT>(s, a.group);
    const long long per = run_length(total, blocks);
    const long long first = before + (static_cast<long long>(h) * groups + r / ROWS) * each;
    const long long c0 = (first + kSetup) / per, c1 = (first + each - 1) / per;
    const int own = static_cast<int>(c1 - c0 + 1);
    pdl_wait();
    if (r >= s.rows * a.group || (own == 1 && a.prefix_len == 0)) return;  // no row; finished by its block
    const size_t row = h * static_cast<size_t>(a.prefix_rows) + static_cast<size_t>(s.row0) * a.group + r;
    const size_t split = static_cast<size_t>(a.n_kv) * a.prefix_rows;
    float y[D / 32] = {};
    join_row<D>(
        -INFINITY, 0.0f, y, own + a.prefix_splits,
        [&](int i, const float2*& ml, const float*& o) {
            if (i >= own) {
                const size_t at = (i - own) * split + row;
                ml = a.prefix_ml + at;
                o = a.prefix_o + at * D;
            } else if (own == 1) {
                ml = a.whole_ml + row;
                o = a.whole_o + row * D;
            } else {
                const size_t at = ((c0 + i) * 2 + (i == 0)) * ROWS + r % ROWS;
                ml = a.own_ml + at;
                o = a.own_o + at * D;
            }
        },
        static_cast<uint16_t*>(a.out) + (s.row0 + token_of(a, r)) * a.out_stride +
            (h * a.group + r - token_of(a, r) * a.group) * D,
        a.f16);
}

template <int D, bool E4M3, int NT, Mode MODE>
void launch_strips(const PagedArgs& a, long long strips, cudaStream_t s) {
    constexpr int bytes = OwnSmem<D, E4M3, NT, MODE>::kBytes;
    auto kernel = own_pages_kernel<D, E4M3, NT, MODE>;
    Q3_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    launch_dep(a.prefix_splits > 0, kernel, dim3(static_cast<unsigned>(strips)),
               dim3(Shape<D, E4M3, NT, MODE>::kWarps * 32), bytes, s, a);
}

template <int D, bool E4M3, int NT>
void launch_own(const PagedArgs& a, int sms, cudaStream_t s) {
    const long long groups = (static_cast<long long>(a.max_q) * a.group + 8 * NT - 1) / (8 * NT);
    const long long strips = static_cast<long long>(a.n_seqs) * a.n_kv * groups;
    if (a.inline_pages > 0 || a.table_stride <= kStripPages) {
        // Short sequences: a block a strip, no line to find and nothing to join after it.
        if (strips <= sms) launch_strips<D, E4M3, NT, kWideStrip>(a, strips, s);
        else launch_strips<D, E4M3, NT, kStrip>(a, strips, s);
        return;
    }
    constexpr int per_sm = Shape<D, E4M3, NT, kLine>::kBlocks, bytes = OwnSmem<D, E4M3, NT, kLine>::kBytes;
    // No more blocks than the table's width could fill.
    const long long most = (strips * (a.table_stride + kSetup) + kMinUnits - 1) / kMinUnits;
    const int grid = static_cast<int>(
        std::min({most, static_cast<long long>(sms) * per_sm, static_cast<long long>(kMaxBlocks)}));
    auto kernel = own_pages_kernel<D, E4M3, NT, kLine>;
    Q3_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    launch_dep(a.prefix_len > 0, kernel, dim3(grid), dim3(kThreads), bytes, s, a);
    const long long rows = static_cast<long long>(a.n_seqs) * a.n_kv * a.max_q * a.group;
    launch_dep(true, join_kernel<D, NT>, dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps)),
               dim3(kThreads), 0, s, a, static_cast<unsigned>(grid));
}

template <int D, bool E4M3>
void launch_own(const PagedArgs& a, int sms, cudaStream_t s) {
    if (a.max_q * a.group <= 8) launch_own<D, E4M3, 1>(a, sms, s);
    else launch_own<D, E4M3, 2>(a, sms, s);
}

// ------------------------------------------------------------------ host

constexpr int kMaxGroup = 64, kMaxRows = 128, kMaxBatchRows = 1 << 23, kMaxPrefix = 1 << 28;
constexpr int kMaxTable = 1 << 26;  // pages: token numbers then stay inside 31 bits

bool sizes_ok(const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs, int max_q, int prefix_len) {
    return n_heads > 0 && n_heads % pool->n_kv_heads == 0 && n_heads / pool->n_kv_heads <= kMaxGroup &&
           n_q >= 0 && n_seqs >= 0 && max_q > 0 &&
           static_cast<long long>(max_q) * (n_heads / pool->n_kv_heads) <= kMaxRows && prefix_len >= 0 && prefix_len <= kMaxPrefix &&
           static_cast<long long>(n_q) * (n_heads / pool->n_kv_heads) <= kMaxBatchRows &&
           static_cast<long long>(n_seqs) * max_q * n_heads <= INT_MAX;
}

// Rows of a strip.
int strip_rows(const PagedArgs& a) { return a.max_q * a.group <= 8 ? 8 : 16; }

// The workspace's arrays begin on multiples of 256 bytes.
size_t whole_lines(size_t bytes) { return (bytes + 255) & ~size_t(255); }

// Lays the workspace out from its start for this call.
void lay_out(PagedArgs& a, uint8_t* base, int head_dim) {
    auto take = [&](size_t bytes) {
        uint8_t* p = base;
        base += whole_lines(bytes);
        return p;
    };
    const size_t rows = strip_rows(a);
    a.own_ml = reinterpret_cast<float2*>(take(kMaxBlocks * 2 * rows * 8));
    a.own_o = reinterpret_cast<float*>(take(kMaxBlocks * 2 * rows * head_dim * 4));
    if (a.prefix_len > 0) {
        a.prefix_rows = a.n_q * a.group;
        const size_t all = static_cast<size_t>(a.n_kv) * a.prefix_rows;
        a.whole_ml = reinterpret_cast<float2*>(take(all * 8));
        a.whole_o = reinterpret_cast<float*>(take(all * head_dim * 4));
        a.prefix_splits = prefix_splits(a.n_kv, a.prefix_rows, a.prefix_len);
        a.prefix_ml = reinterpret_cast<float2*>(take(a.prefix_splits * all * 8));
        a.prefix_o = reinterpret_cast<float*>(take(a.prefix_splits * all * head_dim * 4));
    }
}

// The size that the call, and every call of fewer rows, sequences, rows a sequence or shared tokens, lays out.
size_t workspace_size(const PagedArgs& a, int head_dim) {
    const size_t cell = static_cast<size_t>(head_dim) * 4, rows = strip_rows(a);
    size_t at = whole_lines(kMaxBlocks * 2 * rows * 8) + whole_lines(kMaxBlocks * 2 * rows * cell);
    if (a.prefix_len > 0) {
        const size_t all = static_cast<size_t>(a.n_kv) * a.n_q * a.group;
        const size_t parts = a.n_kv * prefix_part_rows(a.n_kv, a.n_q * a.group, a.prefix_len);
        at += whole_lines(all * 8) + whole_lines(all * cell) + whole_lines(parts * 8) + whole_lines(parts * cell);
    }
    return at;
}

void paged_attention(void* out, void* workspace, const void* q, int type, int64_t q_stride,
                     int64_t out_stride, const q3_kv_pool* pool, int n_heads, int n_q, int n_seqs,
                     int max_q, const int32_t* q_start, const int32_t* kv_len, const int32_t* table,
                     int table_stride, const int32_t* prefix_table, int prefix_len, void* stream) {
    check_pool(pool);
    if (type != Q3_TYPE_BF16 && !(type == Q3_TYPE_F16 && pool->type == Q3_TYPE_E4M3)) {
        throw std::invalid_argument("paged attention: type must be BF16, or F16 with an e4m3 pool");
    }
    if (!sizes_ok(pool, n_heads, n_q, n_seqs, max_q, prefix_len) || table_stride < 0 || table_stride > kMaxTable) {
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
    a.group_magic = a.group == 1 ? 0u : static_cast<unsigned>(((1ull << 32) + a.group - 1) / a.group);
    a.n_q = n_q;
    a.n_seqs = n_seqs;
    a.max_q = max_q;
    a.table_stride = table_stride;
    a.prefix_len = prefix_len;
    a.f16 = type == Q3_TYPE_F16;
    lay_out(a, static_cast<uint8_t*>(workspace), pool->head_dim);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = pool->type == Q3_TYPE_E4M3;
    const int rows = strip_rows(a);
    const long long strips = static_cast<long long>(n_seqs) * a.n_kv * ((max_q * a.group + rows - 1) / rows);
    const long long pages = (prefix_len + kPageTokens - 1LL) / kPageTokens;
    if (pages + table_stride <= kInlinePages && strips * pages <= kInlineWork) {
        a.inline_pages = static_cast<int>(pages);
        a.prefix_splits = 0;
    } else if (prefix_len > 0) {
        launch_prefix_attention(a, pool->head_dim, e4m3, s);
    }
    if (pool->head_dim == 64) {
        e4m3 ? launch_own<64, true>(a, on.sm_count(), s) : launch_own<64, false>(a, on.sm_count(), s);
    } else {
        e4m3 ? launch_own<128, true>(a, on.sm_count(), s) : launch_own<128, false>(a, on.sm_count(), s);
    }
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
    q3::PagedArgs a{};
    a.n_kv = pool->n_kv_heads;
    a.group = n_heads / pool->n_kv_heads;
    a.n_q = n_q;
    a.n_seqs = n_seqs;
    a.max_q = max_q;
    a.prefix_len = prefix_len;
    return q3::workspace_size(a, pool->head_dim);
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
