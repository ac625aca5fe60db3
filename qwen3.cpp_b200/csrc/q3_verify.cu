// q3_verify_drafts: drafted tokens accepted or rejected against the target's probabilities, and the
// token after them drawn, from given uniform numbers.
//
// Draft j (token t, drawn from q_j) is accepted while u_j q_j(t) < p_j(t); after a rejection at j the
// next token comes from max(p_j - q_j, 0), after none from p_n: the tokens are then distributed as if
// all had been drawn from the target. Drawing is the inversion of the running sum. fp32 factors and
// differences are exact in 64 bits, and a running sum over 1.5e5 values is within ~1e-13 there, so the
// drawn token does not hang on the order of the additions.
//
// Only the accepted drafts' single values and one row of p and q are read. A cluster of up to 8 CTAs
// takes a sequence: every CTA finds the accepted count (a few gathers), sums its share of the row, one
// contiguous piece a warp, and passes its sum to the others' shared memory; one cluster barrier later
// each knows the total and the sums before it, and the one warp in whose piece the goal falls goes
// through that piece again (from cache) for the index. One launch, no workspace. Bound by HBM for
// many sequences (2 * vocab * 4 bytes each), by latency for one: TIMES.
#include <algorithm>
#include <climits>

#include "q3_paged.cuh"

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

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxCtas = 8;      // the portable cluster size
constexpr int kLeastShare = 4096;  // values that are worth a CTA: below, its start costs more than it reads

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

template <int V>
__device__ __forceinline__ Piece sum_piece(const Row& row, int i0, int i1) {
    double sum = 0.0;
    int last = -1;
    for_row<V, 4>(row, i0, i1, [&](int i, const double (&r)[V]) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            sum += r[k];
            if (r[k] > 0.0) last = i + k;
        }
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return {sum, static_cast<int>(__reduce_max_sync(0xffffffffu, last))};
}

// First index of [i0, i1) at which the running sum, `before` in front of it, passes goal; `last` if the
// roundings of another order keep it from that.
template <int V>
__device__ __forceinline__ int find_in_piece(const Row& row, int i0, int i1, double before, double goal, int last) {
    int found = INT_MAX;
    const int lane = threadIdx.x & 31;
    for_row<V, 1>(row, i0, i1, [&](int i, const double (&r)[V]) {
        double mine = 0.0;
#pragma unroll
        for (int k = 0; k < V; ++k) mine += r[k];
        double run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += x;
        }
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

__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
    __shared__ Piece warps_s[kVerifyWarps];
    __shared__ Piece ctas_s[2][kMaxCtas];  // written by the cluster's CTAs, per attempt
    __shared__ int accepted_s;
    const int b = blockIdx.x / a.ctas, rank = blockIdx.x % a.ctas;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int32_t* tok = a.draft_tokens + static_cast<size_t>(b) * a.max_drafts;
    int count = a.max_drafts;
    if (a.max_drafts && a.n_drafts) count = min(max(a.n_drafts[b], 0), a.max_drafts);
    if (warp == 0) {
        int n = count;
        for (int j0 = 0; j0 < count; j0 += 32) {
            const int j = j0 + lane;
            bool good = j < count;
            if (good) {
                const int t = tok[j];
                const double u = a.u_accept[static_cast<size_t>(b) * a.max_drafts + j];
                good = t >= 0 && t < a.vocab;
                if (good) {
                    const double p = a.target[b * a.t_seq + j * a.t_row + t];
                    const float q = a.draft ? a.draft[b * a.d_seq + j * a.d_row + t] : 1.0f;
                    good = u * share(q) < p;
                }
            }
            const unsigned bad = __ballot_sync(0xffffffffu, !good);
            if (bad) {
                n = min(n, j0 + __ffs(bad) - 1);
                break;
            }
        }
        if (lane == 0) accepted_s = n;
    }
    __syncthreads();
    const int n = accepted_s;
    Row row;
    row.p = a.target + b * a.t_seq + n * a.t_row;
    row.q = n < count && a.draft ? a.draft + b * a.d_seq + n * a.d_row : nullptr;
    row.one = n < count && !a.draft ? tok[n] : -1;
    // Pieces start on multiples of 4, so that they are as aligned as the row.
    const long long pieces = static_cast<long long>(a.ctas) * kVerifyWarps;
    const int per = static_cast<int>(((a.vocab + pieces - 1) / pieces + 3) / 4 * 4);
    const int i0 = static_cast<int>(min(static_cast<long long>(a.vocab), (rank * kVerifyWarps + warp) * static_cast<long long>(per)));
    const int i1 = static_cast<int>(min(static_cast<long long>(a.vocab), i0 + static_cast<long long>(per)));
    const bool vec = ((reinterpret_cast<uintptr_t>(row.p) | reinterpret_cast<uintptr_t>(row.q)) & 15) == 0;
    Piece mine{};
    double total = 0.0, before = 0.0, after = 0.0;
    int last = -1;
    for (int attempt = 0; attempt < 2; ++attempt) {
        mine = vec ? sum_piece<4>(row, i0, i1) : sum_piece<1>(row, i0, i1);
        if (lane == 0) warps_s[warp] = mine;
        __syncthreads();
        if (tid < a.ctas) {
            Piece all{0.0, -1};
#pragma unroll
            for (int w = 0; w < kVerifyWarps; ++w) {
                all.sum += warps_s[w].sum;
                all.last = max(all.last, warps_s[w].last);
            }
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                         : "=r"(to)
                         : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(&ctas_s[attempt][rank]))), "r"(tid));
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(all.sum) : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 8), "r"(all.last) : "memory");
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        total = before = 0.0;
        last = -1;
        for (int c = 0; c < a.ctas; ++c) {
            if (c == rank) before = total;
            total += ctas_s[attempt][c].sum;
            last = max(last, ctas_s[attempt][c].last);
        }
        // This piece's two ends, added up in one order everywhere, so that one's end is the next one's
        // beginning to the bit and every goal lies in exactly one.
        double in_cta = 0.0;
        for (int w = 0; w < warp; ++w) in_cta += warps_s[w].sum;
        after = before + (in_cta + mine.sum);
        before += in_cta;
        if (total > 0.0) break;
        row.q = nullptr;  // nothing is left over: the target's own row
        row.one = -1;
        __syncthreads();
    }
    const double goal = fmax(static_cast<double>(a.u_sample[b]) * total, 0.0);
    int32_t* out = a.tokens + static_cast<size_t>(b) * (a.max_drafts + 1);
    if (before <= goal && goal < after) {
        const int at = vec ? find_in_piece<4>(row, i0, i1, before, goal, mine.last)
                           : find_in_piece<1>(row, i0, i1, before, goal, mine.last);
        if (lane == 0) out[n] = at;
    }
    if (rank == 0) {
        if (tid == 0) {
            a.n_accepted[b] = n;
            if (!(goal < total)) out[n] = max(last, 0);
        }
        for (int j = tid; j <= a.max_drafts; j += kVerifyThreads) {
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
        if (n_seqs < 0 || max_drafts < 0 || max_drafts > 1024 || vocab <= 0) {
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
        // As many CTAs as have kLeastShare values each, a power of two.
        int ctas = 1;
        while (ctas < q3::kMaxCtas && vocab >= 2 * ctas * q3::kLeastShare) ctas *= 2;
        if (n_seqs > INT_MAX / ctas) throw std::invalid_argument("draft verification: size out of range");
        const q3::VerifyArgs a{tokens, n_accepted, target, draft, draft_tokens, n_drafts, u_accept,
                               u_sample, t_seq, t_row, d_seq, d_row, max_drafts, vocab, ctas};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(n_seqs) * ctas);
        cfg.blockDim = dim3(q3::kVerifyThreads);
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
