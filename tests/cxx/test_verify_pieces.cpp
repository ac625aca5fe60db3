// How verify_kernel cuts a row, followed for every token of many vocabularies: what each thread of a CTA works
// out for itself has to agree, the pieces have to tile the row, and pieces with values start on multiples
// of 4.
#include <cstdio>
#include <initializer_list>

#include "q3_verify_pieces.cuh"

using namespace q3;

static int fail(const char* what, int vocab, int ctas, int warps, int at) {
    std::printf("%s: vocab %d, %d CTAs of %d warps, at %d\n", what, vocab, ctas, warps, at);
    return 1;
}

// `whole` in pieces of `step`, `n` of them: they tile it, and those that hold values are aligned.
static bool tiles(Span whole, int step, int n) {
    int at = whole.i0;
    for (int k = 0; k < n; ++k) {
        const Span p = piece(whole, step, k);
        if (p.i0 != at || p.size() < 0 || p.size() > step) return false;
        if (p.size() > 0 && p.i0 % 4 != 0) return false;
        at = p.i1;
    }
    return at == whole.i1;
}

static int check(int vocab, int ctas, int warps) {
    const int per = piece_step(vocab, ctas * warps);
    const Span row{0, vocab};
    const long long share = static_cast<long long>(per) * warps;
    int at = 0;
    for (int rank = 0; rank < ctas; ++rank) {
        const Span cta = piece(row, share, rank);
        if (cta.i0 != at || cta.size() < 0) return fail("shares do not tile the row", vocab, ctas, warps, rank);
        at = cta.i1;
        if (!tiles(cta, per, warps)) return fail("pieces do not tile a share", vocab, ctas, warps, rank);
        // Every span that the search can come to, down to those that one warp scans.
        struct {
            Span span;
            int step;
        } left[4096];
        int n = 0;
        left[n++] = {cta, per};
        while (n) {
            const auto x = left[--n];
            int covered = x.span.i0;
            for (int k = 0; k < warps; ++k) {
                const Span p = piece(x.span, x.step, k);
                if (p.size() == 0) continue;
                if (p.i0 != covered) return fail("a gap", vocab, ctas, warps, p.i0);
                covered = p.i1;
                if (p.size() <= kScan) continue;
                const int step = piece_step(p.size(), warps);
                if (step >= p.size()) return fail("no progress", vocab, ctas, warps, p.i0);
                if (!tiles(p, step, warps)) return fail("pieces do not tile a piece", vocab, ctas, warps, p.i0);
                if (n == 4096) return fail("too many", vocab, ctas, warps, p.i0);
                left[n++] = {p, step};
            }
            if (covered != x.span.i1) return fail("tokens in no piece", vocab, ctas, warps, covered);
        }
    }
    if (at != vocab) return fail("shares do not tile the row", vocab, ctas, warps, at);
    return 0;
}

int main() {
    const int wanted[] = {1,     2,     3,     4,     5,     127,    128,    129,    511,    512,    8191,      8192,
                          8193,  32768, 50257, 65535, 65536, 81000,  81001,  99999,  128256, 129280, 131071,    131072,
                          151935, 151936, 151937, 200000, 262143, 262144, 1000003, 16777217, (1 << 30) - 1, 1 << 30};
    unsigned seed = 1;
    int vocabs = 0;
    auto all = [&](int vocab) {
        ++vocabs;
        for (const int n_seqs : {1, 4, 5, 8, 18, 19, 64, 300}) {
            const int ctas = verify_ctas(n_seqs, vocab);
            const int warps = verify_threads(n_seqs, ctas, 148) / 32;
            if (ctas < 1 || ctas > kMaxCtas || (ctas & (ctas - 1))) return fail("CTAs", vocab, ctas, warps, n_seqs);
            if (const int bad = check(vocab, ctas, warps)) return bad;
        }
        return 0;
    };
    for (const int v : wanted) {
        if (all(v)) return 1;
    }
    for (int i = 0; i < 400; ++i) {
        seed = seed * 1664525u + 1013904223u;
        if (all(1 + static_cast<int>(seed % 200000u))) return 1;
    }
    std::printf("verify pieces passed: %d vocabularies\n", vocabs);
    return 0;
}
