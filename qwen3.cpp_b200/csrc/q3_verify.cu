// q3_verify_drafts: drafted tokens accepted or rejected against the target's probabilities, and the
// token after them drawn, from given uniform numbers.
//
// Draft j (token t, drawn from q_j) is accepted while u_j q_j(t) < p_j(t); after a rejection at j the
// next token comes from max(p_j - q_j, 0), after none from p_n: the tokens are then distributed as if
// all had been drawn from the target. Drawing is the inversion of the running sum. fp32 factors and
// differences are exact in 64 bits, and a running sum over 1.5e5 values is within ~1e-13 there, so the
// drawn token does not hang on the order of the additions.
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
    int max_drafts, vocab;
};

constexpr int kVerifyThreads = 1024;

__device__ __forceinline__ double share(double x) { return x > 0.0 ? x : 0.0; }  // NaN is 0

__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
    __shared__ double sums[kVerifyThreads];
    __shared__ int accepted_s, found_s, last_s;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int32_t* tok = a.draft_tokens + static_cast<size_t>(b) * a.max_drafts;
    int count = a.max_drafts;
    if (a.max_drafts && a.n_drafts) count = min(max(a.n_drafts[b], 0), a.max_drafts);
    if (tid == 0) {
        int j = 0;
        for (; j < count; ++j) {
            const int t = tok[j];
            if (t < 0 || t >= a.vocab) break;
            const double p = a.target[b * a.t_seq + j * a.t_row + t];
            const double q = a.draft ? a.draft[b * a.d_seq + j * a.d_row + t] : 1.0;
            const double u = a.u_accept[static_cast<size_t>(b) * a.max_drafts + j];
            if (!(u * share(q) < p)) break;
        }
        accepted_s = j;
        found_s = INT_MAX;
        last_s = -1;
    }
    __syncthreads();
    const int n = accepted_s;
    const float* p = a.target + b * a.t_seq + n * a.t_row;
    const float* q = n < count && a.draft ? a.draft + b * a.d_seq + n * a.d_row : nullptr;
    const int certain = n < count && !a.draft ? tok[n] : -1;
    const int per = (a.vocab + kVerifyThreads - 1) / kVerifyThreads;
    const int i0 = min(tid * per, a.vocab), i1 = min(i0 + per, a.vocab);
    bool residual = true;
    double total = 0.0, before = 0.0, mine = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        mine = 0.0;
        for (int i = i0; i < i1; ++i) {
            double x = share(p[i]);
            if (residual) x = share(x - (q ? share(q[i]) : (i == certain ? 1.0 : 0.0)));
            mine += x;
        }
        __syncthreads();
        sums[tid] = mine;
        __syncthreads();
        total = before = 0.0;
        for (int i = 0; i < kVerifyThreads; ++i) {
            if (i == tid) before = total;
            total += sums[i];
        }
        if (total > 0.0) break;
        residual = false;
    }
    const double goal = static_cast<double>(a.u_sample[b]) * total;
    double c = before;
    int last = -1, found = INT_MAX;
    for (int i = i0; i < i1; ++i) {
        double x = share(p[i]);
        if (residual) x = share(x - (q ? share(q[i]) : (i == certain ? 1.0 : 0.0)));
        c += x;
        if (x > 0.0) last = i;
        if (c > goal) {
            found = i;
            break;
        }
    }
    atomicMin(&found_s, found);
    atomicMax(&last_s, last);
    __syncthreads();
    if (tid == 0) a.n_accepted[b] = n;
    const int drawn = found_s != INT_MAX ? found_s : max(last_s, 0);
    for (int j = tid; j <= a.max_drafts; j += kVerifyThreads) {
        a.tokens[static_cast<size_t>(b) * (a.max_drafts + 1) + j] = j < n ? tok[j] : j == n ? drawn : -1;
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
        const q3::VerifyArgs a{tokens, n_accepted, target, draft, draft_tokens, n_drafts, u_accept,
                               u_sample, t_seq, t_row, d_seq, d_row, max_drafts, vocab};
        q3::launch_dep(false, q3::verify_kernel, dim3(n_seqs), dim3(q3::kVerifyThreads), 0,
                       static_cast<cudaStream_t>(stream), a);
    });
}
