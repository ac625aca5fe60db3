// How verify_kernel cuts a row of the vocabulary: plain C++, so that the arithmetic can be checked without
// a GPU.
//
// A row is cut into ctas * warps pieces of `step` values, a CTA's share is the run of its warps' pieces,
// and the piece that the drawn token lies in is cut among the warps again. Everything is worked out from the
// whole that is cut, never from a piece whose start was held back at the whole's end: all threads of a CTA
// then agree on the share, the pieces and the number of rounds, the pieces tile the row, and pieces with
// values in them start on multiples of 4 (a step is one), as aligned as the row.
#pragma once

#ifdef __CUDACC__
#define Q3_PIECES __host__ __device__ __forceinline__
#else
#define Q3_PIECES inline
#endif

namespace q3 {

struct Span {
    int i0, i1;
    Q3_PIECES int size() const { return i1 - i0; }
};

// Values of each of n pieces of `size`.
Q3_PIECES int piece_step(int size, int n) {
    return static_cast<int>(((static_cast<long long>(size) + n - 1) / n + 3) / 4 * 4);
}

// Piece k of `whole` in pieces of `step`: empty past the end.
Q3_PIECES Span piece(Span whole, long long step, int k) {
    const long long i0 = whole.i0 + k * step;
    const long long a = i0 < whole.i1 ? i0 : whole.i1;
    return {static_cast<int>(a), static_cast<int>(a + step < whole.i1 ? a + step : whole.i1)};
}

constexpr int kVerifyThreads = 512;  // at most
constexpr int kMaxCtas = 16;         // of a cluster
constexpr int kLeastShare = 4096;    // values that are worth a CTA: below, its start costs more than it reads
constexpr int kScan = 128;           // values that one warp scans

// CTAs of a sequence: as many as have kLeastShare values each, a power of two: up to 16 for up to 4 sequences
// (a multiprocessor reads about 40 GB/s from L2, so one sequence's row takes 7.1 us on 16 and 8.3 on 8), else
// up to 8 (clusters of 16 find room less easily: 64 sequences 36 us against 24).
Q3_PIECES int verify_ctas(int n_seqs, int vocab) {
    const int most = n_seqs <= 4 ? kMaxCtas : kMaxCtas / 2;
    int ctas = 1;
    while (ctas < most && vocab >= 2 * ctas * kLeastShare) ctas *= 2;
    return ctas;
}

// Threads of a CTA. With more CTAs than multiprocessors smaller ones, so that they are all resident at once
// (64 sequences: 24 us against 28); else the larger, whose lanes go round less often.
Q3_PIECES int verify_threads(int n_seqs, int ctas, int sms) {
    return static_cast<long long>(n_seqs) * ctas > sms ? kVerifyThreads / 2 : kVerifyThreads;
}

}  // namespace q3
