// Newton-Schulz orthogonalisation and the Muon step: shared types, and the host-side plan of a call.
//
// For an update U (rows x cols), X = U or U^T so that X is m x n with m <= n:
//
//   X_0 = U / max(||U||_F, eps);   A = X X^T;   P = b A + c A A;   X <- a X + P X      (`steps` times)
//
// Three matrix products a step, all on the matrix cores with 16-bit operands and 32-bit sums. An fp32 value v is held
// as two fp16 numbers v * scale = hi + lo (22 bits); a product of two such values is hi hi + hi lo + lo hi. The scales
// are fixed powers of two (below): X stays below 4 and P below 12 in the 2-norm, which the host checks for the
// coefficients of the call, so every entry of X, A and P is in range and its lo part far above fp16's smallest step.
//
// The Muon step wraps it:  B += (1 - mu)(G - B);  U = G + mu (B - G) (Nesterov) or B;  O = orthogonalised U;
//                          W = W decay - alpha O,   decay = 1 - lr weight_decay, alpha = lr * (a factor of the shape)
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <vector>

namespace pccl::kernels {

constexpr float kMuonScaleX = 8192.0f; // entries of X:  |x| <= 4     -> 32768 (fp16 holds 65504)
constexpr float kMuonScaleA = 1024.0f; // entries of A:  |a| <= 4^2   -> 16384
constexpr float kMuonScaleP = 4096.0f; // entries of P:  |p| <= 12    -> 49152
constexpr int kMuonPad = 64;           // X, A and P are padded to this with zeros, which the iteration keeps zero
constexpr int kMuonMaxMats = 48;       // entries of one launch (they travel in the kernel arguments)
constexpr int kMuonMaxSmall = 1 << 21;  // matrices of one workgroup in a launch, which has fewer than 2^32 threads
constexpr int kMuonMaxPartials = 512;  // partial sums of squares of one matrix
constexpr int kMuonPrepBlock = 4096;   // elements one workgroup of the first pass takes at least
constexpr size_t kMuonWorkspaceBudget = size_t(4) << 30; // matrices are taken in groups of at most this (or one)

// `count` matrices of one shape, one after the other in memory (contiguous, row-major)
struct MuonEntry {
    const void *g = nullptr; // gradient (or the matrix to orthogonalise)
    void *w = nullptr;       // parameter (or the result)
    float *mom = nullptr;    // momentum buffer; nullptr: orthogonalise g
    float alpha = 0.0f;
    int rows = 0, cols = 0, count = 0;
    int mp = 0, np = 0;   // padded smaller / larger side
    int partials = 0;     // workgroups of the first pass per matrix
    size_t off = 0;       // bytes into the workspace, first matrix of the entry
};

struct MuonParams {
    int steps = 5;
    float a = 3.4445f, b = -4.7750f, c = 2.0315f;
    double eps = 1e-7;
    float momentum = 0.95f;
    float decay = 1.0f;
    int nesterov = 1;
};

// workspace of one matrix: X hi, lo twice (a step reads one and writes the other), A hi, lo, P hi, lo, partial sums
inline size_t muon_matrix_bytes(int mp, int np) {
    return 2 * (4 * static_cast<size_t>(mp) * np + 4 * static_cast<size_t>(mp) * mp) + kMuonMaxPartials * sizeof(double);
}

// matrices whose X, A and P one workgroup holds in LDS (160 KB): they need no workspace
inline bool muon_fits_lds(int mp, int np) { return (mp == 64 && np <= 256) || (mp == 128 && np == 128); }

inline int muon_pad(int64_t v) { return static_cast<int>((v + kMuonPad - 1) / kMuonPad * kMuonPad); }

// Splits the entries into groups that run one after the other in the same workspace; returns the workspace's size.
inline size_t muon_plan(const std::vector<MuonEntry> &entries, size_t esize_g, size_t esize_w,
                        std::vector<std::vector<MuonEntry>> *groups) {
    size_t need = 0, used = 0, small = 0; // small: matrices of the group that fit in LDS
    std::vector<MuonEntry> group;
    const auto flush = [&] {
        if (group.empty()) return;
        need = std::max(need, used);
        if (groups) groups->push_back(group);
        group.clear();
        used = small = 0;
    };
    for (MuonEntry e : entries) {
        if (e.count == 0 || e.rows == 0 || e.cols == 0) continue;
        e.mp = muon_pad(std::min(e.rows, e.cols));
        e.np = muon_pad(std::max(e.rows, e.cols));
        const size_t elems = static_cast<size_t>(e.rows) * e.cols;
        const size_t bytes = muon_fits_lds(e.mp, e.np) ? 0 : muon_matrix_bytes(e.mp, e.np);
        e.partials = static_cast<int>(
            std::min<size_t>(kMuonMaxPartials, (elems + kMuonPrepBlock - 1) / kMuonPrepBlock));
        int left = e.count;
        while (left > 0) {
            size_t room = kMuonMaxSmall - small;
            if (bytes > 0) room = used < kMuonWorkspaceBudget ? (kMuonWorkspaceBudget - used) / bytes : 0;
            if ((room == 0 && (used > 0 || bytes == 0)) || static_cast<int>(group.size()) == kMuonMaxMats) {
                flush();
                continue;
            }
            MuonEntry part = e;
            part.count = static_cast<int>(std::min<size_t>(left, std::max<size_t>(room, 1)));
            part.off = used;
            group.push_back(part);
            used += bytes * part.count;
            small += bytes == 0 ? part.count : 0;
            left -= part.count;
            e.g = static_cast<const uint8_t *>(e.g) + esize_g * elems * part.count;
            e.w = static_cast<uint8_t *>(e.w) + esize_w * elems * part.count;
            if (e.mom) e.mom += elems * part.count;
        }
    }
    flush();
    return need;
}

} // namespace pccl::kernels
