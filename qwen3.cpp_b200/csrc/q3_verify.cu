// q3_verify_drafts: drafted tokens accepted or rejected against the target's probabilities, and the
// token after them drawn, from given uniform numbers.
//
// Draft j (token t, drawn from q_j) is accepted while u_j q_j(t) < p_j(t); after a rejection at j the
// next token comes from max(p_j - q_j, 0), after none from p_n: the tokens are then distributed as if
// all had been drawn from the target. Drawing is the inversion of the running sum. fp32 factors and
// differences are exact in 64 bits, and a running sum over 1.5e5 values is within ~1e-13 there, so the
// drawn token does not hang on the order of the additions.
//
// Only the accepted drafts' single values and one row of p and q are read. A cluster of up to 16 CTAs
// takes a sequence: every CTA finds the accepted count (a few gathers), sums its share of the row, one
// contiguous piece a warp, and passes its sum to the others' shared memory; one cluster barrier later
// each knows the total and the sums before it, and the one warp in whose piece the goal falls goes
// through that piece again (from cache) for the index. One launch, no workspace. With vocab 151936, 64
// sequences of 5 drafts take 24 us (78 MB, 3.2 TB/s: 14 us of them the reading, the rest the chain of
// dependent steps around it), one of 4 drafts 7.1 us, all latency.
#include <algorithm>
#include <climits>

#include "q3_paged.cuh"
#include "q3_verify_pieces.cuh"

namespace q3 {

namespace {

struct VerifyArgs {
    int32_t* tokens;
    int32_t* n_accepted;
    const float* target;
    const float* draft;
    const int32_t* draft_tokens;
    const int32_t* n_drafts;
    const float* u_accept;
    const float* u_sample;
    long long t_seq, t_row, d_seq, d_row;
    int max_drafts, vocab, ctas;  // ctas: of a sequence's cluster
};

constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kUnroll = 2;  // 16-byte loads of p, and of q, that a lane has on their way (5: 6% slower)

__device__ __forceinline__ float share(float x) { return x > 0.0f ? x : 0.0f; }  // NaN is 0

struct Piece {
    double sum;
    int last;  // last index with a positive share, -1 for none
};

// The row that the token is drawn from: max(p - q, 0), q given (one = -1), certain for token `one`
// (q null), or nothing (q null, one = -1).
struct Row {
    const float* p;
    const float* q;
    int one;
    __device__ __forceinline__ double at(float x, float y, int i) const {
        if (!q) y = i == one ? 1.0f : 0.0f;
        x = share(x);
        y = share(y);
        return x > y ? static_cast<double>(x) - static_cast<double>(y) : 0.0;
    }
};

// Calls f(i, value) for this lane's values of [i0, i1), a block of 32 * V after the other, V
// neighbours a lane; UNROLL blocks are loaded before the first is used. f gets each block's values of
// the lane at once: f(first index, value[V]).
template <int V, int UNROLL, typename F>
__device__ __forceinline__ void for_row(const Row& row, int i0, int i1, F f) {
    const int lane = threadIdx.x & 31;
    for (int i = i0; i < i1; i += 32 * V * UNROLL) {
        float x[UNROLL][V], y[UNROLL][V];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int at = i + (u * 32 + lane) * V;
            if constexpr (V == 4) {
                const bool in = at + V <= i1;
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
                if (in) {
                    a = __ldg(reinterpret_cast<const float4*>(row.p + at));
                    if (row.q) b = __ldg(reinterpret_cast<const float4*>(row.q + at));
                } else if (at < i1) {
                    float* pa = &a.x;
                    float* pb = &b.x;
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        if (at + k < i1) {
                            pa[k] = __ldg(row.p + at + k);
                            if (row.q) pb[k] = __ldg(row.q + at + k);
                        }
                    }
                }
                x[u][0] = a.x; x[u][1] = a.y; x[u][2] = a.z; x[u][3] = a.w;
                y[u][0] = b.x; y[u][1] = b.y; y[u][2] = b.z; y[u][3] = b.w;
            } else {
                x[u][0] = at < i1 ? __ldg(row.p + at) : 0.0f;
                y[u][0] = at < i1 && row.q ? __ldg(row.q + at) : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            double r[V];
            const int at = i + (u * 32 + lane) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) r[k] = row.at(x[u][k], y[u][k], at + k);
            f(at, r);
        }
    }
}

// Sum and last share of [i0, i1), for all lanes of the warp. V sums at once: a 64-bit addition takes
// tens of cycles.
template <int V, int UNROLL>
__device__ __forceinline__ Piece sum_piece(const Row& row, int i0, int i1) {
    double part[V] = {};
    int last = -1;
    for_row<V, UNROLL>(row, i0, i1, [&](int i, const double (&r)[V]) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            part[k] += r[k];
            if (r[k] > 0.0) last = i + k;
        }
    });
    double sum = V == 4 ? (part[0] + part[1 % V]) + (part[2 % V] + part[3 % V]) : part[0];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return {sum, static_cast<int>(__reduce_max_sync(0xffffffffu, last))};
}

// The lanes' running sum.
__device__ __forceinline__ double running_sum(double x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// First index of [i0, i1), at most kScan values, at which the running sum, `before` in front of it,
// passes goal; `last` if the roundings of another order keep it from that.
template <int V>
__device__ __forceinline__ int scan(const Row& row, int i0, int i1, double before, double goal, int last) {
    int found = INT_MAX;
    for_row<V, 1>(row, i0, i1, [&](int i, const double (&r)[V]) {
        const double mine = V == 4 ? (r[0] + r[1 % V]) + (r[2 % V] + r[3 % V]) : r[0];
        const double run = running_sum(mine);
        double c = before + (run - mine);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            c += r[k];
            if (r[k] > 0.0 && c > goal) found = min(found, i + k);
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    });
    found = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(found)));
    return found == INT_MAX ? last : found;
}

__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const VerifyArgs a) {
    __shared__ Piece warps_s[kVerifyWarps];
    __shared__ Piece ctas_s[2][kMaxCtas];  // written by the cluster's CTAs, per attempt
    __shared__ int accepted_s;
    const int b = blockIdx.x / a.ctas, rank = blockIdx.x % a.ctas;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n_warps = blockDim.x >> 5;
    // Another CTA's shared memory may be written once that CTA has started: waited for in front of the writes.
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int32_t* tok = a.draft_tokens + static_cast<size_t>(b) * a.max_drafts;
    int count = a.max_drafts;
    if (a.max_drafts && a.n_drafts) count = a.n_drafts[b];
    const float u_sample = a.u_sample[b];  // needed last, on its way first
    if (warp == 0) {
        int n = INT_MAX;
        for (int j0 = 0; j0 < a.max_drafts && n == INT_MAX; j0 += 32) {
            const int j = min(j0 + lane, a.max_drafts - 1);
            const int t = tok[j];  // on its way with the count
            const double u = a.u_accept[static_cast<size_t>(b) * a.max_drafts + j];
            bool good = j0 + lane < min(count, a.max_drafts);
            if (good && t >= 0 && t < a.vocab) {
                const double p = a.target[b * a.t_seq + j * a.t_row + t];
                const float q = a.draft ? a.draft[b * a.d_seq + j * a.d_row + t] : 1.0f;
                good = u * share(q) < p;
            } else {
                good = false;
            }
            const unsigned bad = __ballot_sync(0xffffffffu, !good);
            if (bad) n = j0 + __ffs(bad) - 1;
        }
        n = min(n, a.max_drafts);
        if (lane == 0) accepted_s = n;
    }
    __syncthreads();
    count = min(max(count, 0), a.max_drafts);
    const int n = accepted_s;
    Row row;
    row.p = a.target + b * a.t_seq + n * a.t_row;
    row.q = n < count && a.draft ? a.draft + b * a.d_seq + n * a.d_row : nullptr;
    row.one = n < count && !a.draft ? tok[n] : -1;
    // This CTA's share of the row, the same in all its threads, and this warp's piece of it.
    const int per = piece_step(a.vocab, a.ctas * n_warps);
    const Span cta = piece({0, a.vocab}, static_cast<long long>(per) * n_warps, rank);
    const Span own = piece(cta, per, warp);
    const bool vec = ((reinterpret_cast<uintptr_t>(row.p) | reinterpret_cast<uintptr_t>(row.q)) & 15) == 0;
    // The sums before this CTA's share and up to its end, added up in one order everywhere, so that one's
    // end is the next one's beginning to the bit and every goal lies in exactly one.
    double total = 0.0, cta_before = 0.0, cta_after = 0.0;
    int last = -1;
    for (int attempt = 0; attempt < 2; ++attempt) {
        const Piece mine = vec ? sum_piece<4, kUnroll>(row, own.i0, own.i1) : sum_piece<1, kUnroll>(row, own.i0, own.i1);
        if (lane == 0) warps_s[warp] = mine;
        if (attempt == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        __syncthreads();
        if (warp == 0) {
            Piece all{0.0, -1};
            if (lane < n_warps) all = warps_s[lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all.sum += __shfl_xor_sync(0xffffffffu, all.sum, o);
            all.last = __reduce_max_sync(0xffffffffu, all.last);
            if (lane < a.ctas) {
                uint32_t to;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                             : "=r"(to)
                             : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(&ctas_s[attempt][rank]))), "r"(lane));
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(all.sum) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 8), "r"(all.last) : "memory");
            }
            __syncwarp();
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        total = 0.0;
        last = -1;
        for (int c = 0; c < a.ctas; ++c) {
            if (c == rank) cta_before = total;
            total += ctas_s[attempt][c].sum;
            if (c == rank) cta_after = total;
            last = max(last, ctas_s[attempt][c].last);
        }
        if (total > 0.0) break;
        row.q = nullptr;  // nothing is left over: the target's own row
        row.one = -1;
        __syncthreads();
    }
    const double goal = fmax(static_cast<double>(u_sample) * total, 0.0);
    int32_t* out = a.tokens + static_cast<size_t>(b) * (a.max_drafts + 1);
    if (cta_before <= goal && goal < cta_after) {
        // The token lies in this CTA's share: its warps cut the warp's piece it lies in among them until
        // one warp can scan what is left (one round for 1e5 values). The span that is cut is the same in every
        // thread, so all leave in the same round.
        Span span = cta;
        int step = per;
        double base = cta_before;
        int at = -1;
        while (true) {
            // The piece among the span's that the goal lies in; the last with a share if roundings put it
            // behind all of them. Every warp works it out, a lane a piece.
            Piece x{0.0, -1};
            if (lane < n_warps) x = warps_s[lane];
            const double up_to = running_sum(x.sum);
            const unsigned has = __ballot_sync(0xffffffffu, x.last >= 0);
            const unsigned past = __ballot_sync(0xffffffffu, x.last >= 0 && goal < base + up_to);
            const int pick = past ? __ffs(past) - 1 : 31 - __clz(has | 1u);
            const int pick_last = __shfl_sync(0xffffffffu, x.last, pick);
            const double below = __shfl_sync(0xffffffffu, base + (up_to - x.sum), pick);
            span = piece(span, step, pick);
            base = below;
            if (span.size() <= kScan) {
                if (warp == 0) {
                    at = vec ? scan<4>(row, span.i0, span.i1, base, goal, pick_last)
                             : scan<1>(row, span.i0, span.i1, base, goal, pick_last);
                }
                break;
            }
            step = piece_step(span.size(), n_warps);
            const Span sub = piece(span, step, warp);
            const Piece mine = vec ? sum_piece<4, 1>(row, sub.i0, sub.i1) : sum_piece<1, 4>(row, sub.i0, sub.i1);
            __syncthreads();
            if (lane == 0) warps_s[warp] = mine;
            __syncthreads();
        }
        if (tid == 0) out[n] = at;
    }
    if (rank == 0) {
        if (tid == 0) {
            a.n_accepted[b] = n;
            if (!(goal < total)) out[n] = max(last, 0);
        }
        for (int j = tid; j <= a.max_drafts; j += blockDim.x) {
            if (j != n) out[j] = j < n ? tok[j] : -1;
        }
    }
}

}  // namespace

}  // namespace q3

extern "C" q3_status q3_verify_drafts(int32_t* tokens, int32_t* n_accepted, const float* target,
                                      int64_t t_seq, int64_t t_row, const float* draft, int64_t d_seq,
                                      int64_t d_row, const int32_t* draft_tokens,
                                      const int32_t* n_drafts, const float* u_accept,
                                      const float* u_sample, int n_seqs, int max_drafts, int vocab,
                                      void* stream) {
    return q3::guard([&] {
        if (n_seqs < 0 || max_drafts < 0 || max_drafts > 1024 || vocab <= 0 || vocab > (1 << 30)) {
            throw std::invalid_argument("draft verification: size out of range");
        }
        if (n_seqs == 0) return;
        if (!tokens || !n_accepted || !target || !u_sample ||
            (max_drafts > 0 && (!draft_tokens || !u_accept))) {
            throw std::invalid_argument("draft verification: null pointer");
        }
        if (max_drafts == 0) draft = nullptr;
        if (t_row < vocab || t_seq < 0 || (draft && (d_row < vocab || d_seq < 0))) {
            throw std::invalid_argument("draft verification: stride below the vocabulary");
        }
        for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(n_accepted),
                              static_cast<const void*>(target), static_cast<const void*>(draft),
                              static_cast<const void*>(draft_tokens), static_cast<const void*>(n_drafts),
                              static_cast<const void*>(u_accept), static_cast<const void*>(u_sample)}) {
            if (!q3::aligned(p, 4)) throw std::invalid_argument("draft verification: misaligned pointer");
        }
        const q3::OnDevice on({tokens, n_accepted, target, draft, max_drafts ? draft_tokens : nullptr,
                               n_drafts, max_drafts ? u_accept : nullptr, u_sample});
        const int ctas = q3::verify_ctas(n_seqs, vocab);
        if (n_seqs > INT_MAX / ctas) throw std::invalid_argument("draft verification: size out of range");
        const q3::VerifyArgs a{tokens, n_accepted, target, draft, draft_tokens, n_drafts, u_accept,
                               u_sample, t_seq, t_row, d_seq, d_row, max_drafts, vocab, ctas};
        if (ctas > 8) {
            Q3_CUDA(cudaFuncSetAttribute(q3::verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(n_seqs) * ctas);
        cfg.blockDim = dim3(static_cast<unsigned>(q3::verify_threads(n_seqs, ctas, on.sm_count())));
        cfg.stream = static_cast<cudaStream_t>(stream);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        Q3_CUDA(cudaLaunchKernelEx(&cfg, q3::verify_kernel, a));
    });
}
