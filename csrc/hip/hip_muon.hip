// Newton-Schulz orthogonalisation and the Muon step (formulas, number formats and plan: csrc/kernels/muon_common.hpp).
//
// All matrices of a call, of whatever shapes, go through each stage in one launch: a workgroup finds its matrix and
// tile from its index. Stages: momentum and sums of squares; X_0 in two fp16 parts, padded, on its shorter side; then
// per step A = X X^T and P = b A + c A A over the tiles on and above the diagonal (both halves are written), and
// a X + P X, whose last pass updates the caller's parameters instead of writing X. No atomics and a fixed order of
// every sum: equal calls give equal bits, which the peers of a run rely on.
//
// Every product is three of the 16-bit parts, the error of fp32 products, whatever the type of the result and whatever
// else the call holds. (With one product of the hi parts for A and P X a bf16 result takes 0.5 to 0.7 of the time, but is
// then up to 1.4 times as far off as its own rounding.)
#include <algorithm>

#include "dispatch.hpp"
#include "launchers.hpp"

namespace pccl::hipk {

using kernels::kMuonMaxMats;
using kernels::kMuonMaxPartials;
using kernels::kMuonScaleA;
using kernels::kMuonScaleP;
using kernels::kMuonScaleX;
using kernels::MuonEntry;
using kernels::MuonParams;

namespace {

using half8 = _Float16 __attribute__((ext_vector_type(8)));
using half4 = _Float16 __attribute__((ext_vector_type(4)));
using short4v = short __attribute__((ext_vector_type(4)));
using float16v = float __attribute__((ext_vector_type(16)));

struct MuonTable {
    uint8_t *ws;
    int n;
    int first[kMuonMaxMats]; // first workgroup of each entry in this launch
    MuonEntry e[kMuonMaxMats];
};
static_assert(sizeof(MuonTable) < 4000, "kernel arguments");

// entry of workgroup `b`: the lanes compare one entry each
__device__ __forceinline__ int entry_of(const MuonTable &t, int b) {
    if (t.n == 1) return 0;
    const int lane = threadIdx.x & 63;
    const bool before = lane < t.n && t.first[lane < t.n ? lane : 0] <= b;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
}

// One matrix in the workspace. X, A and P lie in panels of 16 columns, 64 bytes a row [16 hi | 16 lo], all rows of a
// panel one after the other, so that a tile's share of a panel is contiguous.
struct Planes {
    _Float16 *x0, *x1, *a, *p;
    double *part;
};
__device__ __forceinline__ size_t panel_at(int rows, int r, int c) { // of the hi part; the lo part is kLo further
    return (static_cast<size_t>(c >> 4) * rows + r) * 32 + (c & 15);
}
constexpr int kLo = 16;
__device__ __forceinline__ Planes planes_of(uint8_t *ws, const MuonEntry &e, int which) {
    Planes q;
    const size_t xs = static_cast<size_t>(e.mp) * e.np, as = static_cast<size_t>(e.mp) * e.mp; // elements of X, of A
    const size_t bytes = 2 * (4 * xs + 4 * as) + kMuonMaxPartials * sizeof(double);
    uint8_t *base = ws + e.off + bytes * which;
    q.x0 = reinterpret_cast<_Float16 *>(base);
    q.x1 = q.x0 + 2 * xs;
    q.a = q.x1 + 2 * xs;
    q.p = q.a + 2 * as;
    q.part = reinterpret_cast<double *>(q.p + 2 * as);
    return q;
}

template<DType D>
struct Elem;
template<>
struct Elem<DType::F32> {
    using S = float;
};
template<>
struct Elem<DType::BF16> {
    using S = __bf16;
};
template<>
struct Elem<DType::F16> {
    using S = _Float16;
};

// neighbouring elements at any element alignment (parameters are often views into one flat buffer)
template<typename S, int N>
struct __attribute__((packed, aligned(sizeof(S)))) Run {
    S v[N];
};

// sum over a workgroup of 256 in a fixed order, the same in every thread
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double w[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
    __syncthreads();
    return (w[0] + w[1]) + (w[2] + w[3]);
}

// v = hi + lo, N values: one packed conversion for two, and one mixed-precision subtraction (exact) for each
template<int N>
__device__ __forceinline__ void split_fp16(const float (&v)[N], _Float16 __attribute__((ext_vector_type(N))) & hi,
                                           _Float16 __attribute__((ext_vector_type(N))) & lo) {
    using half2v = _Float16 __attribute__((ext_vector_type(2)));
    using float2v = float __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        const half2v h = __builtin_convertvector((float2v{v[k], v[k + 1]}), half2v);
        const float2v r = {__builtin_fmaf(static_cast<float>(h.x), -1.0f, v[k]),
                           __builtin_fmaf(static_cast<float>(h.y), -1.0f, v[k + 1])};
        const half2v l = __builtin_convertvector(r, half2v);
        hi[k] = h.x;
        hi[k + 1] = h.y;
        lo[k] = l.x;
        lo[k + 1] = l.y;
    }
}
__device__ __forceinline__ float join_fp16(_Float16 hi, _Float16 lo) {
    return __builtin_fmaf(static_cast<float>(hi), 1.0f, static_cast<float>(lo));
}

__device__ __forceinline__ float update_of(float g, float m, const MuonParams &p) {
    return p.nesterov ? g + p.momentum * (m - g) : m;
}

} // namespace

// B += (1 - mu)(G - B), and the squares of U summed in 64 bits (a gradient's squares leave fp32's range long before
// the gradient does). Memory bound: 59 M fp32 elements 117 us, 6.0 TB/s.
template<DType G>
__global__ __launch_bounds__(256) void k_muon_momentum(MuonTable t, MuonParams p) {
    using S = typename Elem<G>::S;
    const int i = entry_of(t, blockIdx.x);
    const MuonEntry &e = t.e[i];
    const int b = blockIdx.x - t.first[i], which = b / e.partials, part = b % e.partials;
    const size_t elems = static_cast<size_t>(e.rows) * e.cols;
    const S *g = static_cast<const S *>(e.g) + elems * which;
    float *m = e.mom ? e.mom + elems * which : nullptr;
    const size_t per = (elems + e.partials - 1) / e.partials;
    const size_t s0 = per * part, s1 = s0 + per < elems ? s0 + per : elems;
    double sum = 0.0;
    const auto one = [&](S gv, float &mv) {
        float u = static_cast<float>(gv);
        if (m) {
            mv = mv + (1.0f - p.momentum) * (u - mv);
            u = update_of(u, mv, p);
        }
        sum += static_cast<double>(u) * u;
    };
    size_t k = s0 + threadIdx.x * 4;
    for (; k + 3 * 1024 + 4 <= s1; k += 4 * 1024) { // 4 x 4 elements in flight
        Run<S, 4> gv[4];
        Run<float, 4> mv[4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            gv[j] = *reinterpret_cast<const Run<S, 4> *>(g + k + j * 1024);
            if (m) mv[j] = *reinterpret_cast<const Run<float, 4> *>(m + k + j * 1024);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float v = mv[j].v[x];
                one(gv[j].v[x], v);
                mv[j].v[x] = v;
            }
            if (m) *reinterpret_cast<Run<float, 4> *>(m + k + j * 1024) = mv[j];
        }
    }
    for (; k < s1; k += 1024)
        for (size_t j = k; j < k + 4 && j < s1; ++j) {
            float v = m ? m[j] : 0.0f;
            one(g[j], v);
            if (m) m[j] = v;
        }
    sum = block_sum(sum);
    if (threadIdx.x == 0) planes_of(t.ws, e, which).part[part] = sum;
}

// X_0 = U scale / max(||U||, eps) in two fp16 parts, 64 x 64 tiles, by way of LDS: it is read along the rows of U and
// written in the order of the panels, and a tall U is transposed between. Memory bound: 59 M fp32 elements 143 us,
// 5.0 TB/s (190 us with 16 columns of one row per thread and no LDS).
template<DType G>
__global__ __launch_bounds__(256) void k_muon_start(MuonTable t, MuonParams p) {
    using S = typename Elem<G>::S;
    __shared__ float tile[64][65];
    const int i = entry_of(t, blockIdx.x);
    const MuonEntry &e = t.e[i];
    const int tn = e.np / 64, tiles = e.mp / 64 * tn;
    const int b = blockIdx.x - t.first[i], which = b / tiles, m0 = b % tiles / tn * 64, n0 = b % tiles % tn * 64;
    const Planes q = planes_of(t.ws, e, which);
    const size_t elems = static_cast<size_t>(e.rows) * e.cols;
    const S *g = static_cast<const S *>(e.g) + elems * which;
    const float *mom = e.mom ? e.mom + elems * which : nullptr;
    const bool flip = e.rows > e.cols;
    // a wave reads 4 runs of 64 neighbours of U's rows at a time
    const int c = (threadIdx.x & 15) * 4, uc = (flip ? m0 : n0) + c;
    Run<S, 4> gv[4] = {};
    Run<float, 4> mv[4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int ur = (flip ? n0 : m0) + (threadIdx.x >> 4) + 16 * k;
        const size_t at = static_cast<size_t>(ur) * e.cols + uc;
        if (ur < e.rows && uc + 4 <= e.cols) {
            gv[k] = *reinterpret_cast<const Run<S, 4> *>(g + at);
            if (mom) mv[k] = *reinterpret_cast<const Run<float, 4> *>(mom + at);
        } else if (ur < e.rows) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (uc + j < e.cols) {
                    gv[k].v[j] = g[at + j];
                    if (mom) mv[k].v[j] = mom[at + j];
                }
        }
    }
    double sum = 0.0; // while they are on their way
    for (int k = threadIdx.x; k < e.partials; k += 256) sum += q.part[k];
    sum = block_sum(sum);
    const double norm = sqrt(sum);
    const double scale = static_cast<double>(kMuonScaleX) / (norm > p.eps || norm != norm ? norm : p.eps);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = (threadIdx.x >> 4) + 16 * k;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float u = static_cast<float>(gv[k].v[j]);
            const float v = static_cast<float>((mom ? update_of(u, mv[k].v[j], p) : u) * scale);
            (flip ? tile[c + j][r] : tile[r][c + j]) = v;
        }
    }
    __syncthreads();
    // 16-byte pieces in the order in which they lie in X: 64 bytes of a row, then the next row
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = (threadIdx.x >> 2) & 63, piece = threadIdx.x & 3;
        const bool low = piece & 2;
        const int x = 16 * k + 8 * (piece & 1);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[r][x + j];
        half8 hi, lo;
        split_fp16<8>(v, hi, lo);
        _Float16 *to = q.x0 + panel_at(e.mp, m0 + r, n0 + x) + (low ? kLo : 0);
        *reinterpret_cast<half8 *>(to) = low ? lo : hi;
    }
}

enum { kGram = 0, kPoly = 1, kApply = 2, kFinal = 3 };

struct MuonStage {
    int cur; // which X is read
    float a, b, c, decay;
};

template<int N>
__device__ __forceinline__ void wait_loads() { // all but the N newest loads of this wave have landed, its LDS reads too
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// the same with N per tile and `tiles` < LEFT tiles still allowed to be on their way
template<int N, int LEFT>
__device__ __forceinline__ void wait_tiles(int tiles) {
    if constexpr (LEFT > 0) {
        if (tiles >= LEFT - 1)
            wait_loads<N * (LEFT - 1)>();
        else
            wait_tiles<N, LEFT - 1>(tiles);
    }
}
// orders LDS accesses between the lanes of one wave
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

__device__ __forceinline__ uint32_t lds_offset(const uint8_t *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) uint8_t *)p));
}

// 16 bytes a lane from memory to LDS, 1 KB from `to` on. In assembly, so that the compiler does not make the transposing
// reads of one tile wait for the tiles that are still on their way; the waits are this file's own (wait_tiles).
__device__ __forceinline__ void load_to_lds(const _Float16 *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n"
                 "s_nop 0\n"
                 "global_load_lds_dwordx4 %1, off" ::"s"(to),
                 "v"(from)
                 : "memory", "m0");
}

// N-side fragments of kApply: at[z][s] is where this lane's part of the 4 x 16 block z of piece s lies, column block 1
// lies YSTEP bytes further
template<int NT, int YSTEP>
__device__ __forceinline__ void read_transposed(const uint8_t *base, const uint32_t (&at)[2][2], half8 (&f)[NT][2]) {
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            half4 h[2];
#pragma unroll
            for (int z = 0; z < 2; ++z)
                h[z] = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                     (__attribute__((address_space(3))) short4v *)(base + at[z][s] + y * YSTEP)));
            f[y][s] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
}

// 16-byte pieces of a panel's 64-byte rows trade places in LDS: a fragment's 16-byte reads are served 16 rows at a time
// from 64 banks, so rows 4 apart must differ; the transposing read takes 4 rows of two column blocks at a time, and
// where these lie in two panels their pieces must differ too.
__device__ __forceinline__ int swizzle(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int swizzle(int r, int panel) { return swizzle(r) ^ ((panel & 1) << 1); }

// Work item of this workgroup. Workgroups go to the 8 chiplets in turn; each gets runs of neighbouring tiles, which share
// operands in its L2, and the runs advance together, because the items are sorted by falling length. What the L2s miss
// is what bounds these kernels apart from their products. A run of P X is kBand rows of tiles and as many columns.
constexpr int kBand = 8;
template<int kRun>
__device__ __forceinline__ int place_of_block() {
    const int b = blockIdx.x, n = gridDim.x, window = 8 * kRun;
    const int base = b / window * window, run = n - base < window ? (n - base) / 8 : kRun;
    const int k = b - base;
    return k < 8 * run ? base + (k & 7) * run + (k >> 3) : b;
}

// One product stage. A workgroup computes BM x BN of it. The M side's rows (of X, A or P) lie along the sum, and so do
// the N side's of kGram and kPoly, which multiply by a transpose; kApply's and kFinal's N side is X itself, whose
// fragments are transposed on their way out of LDS. Both sides travel straight to LDS, a panel of the sum at a time.
// The MFMA's first operand is the N side: a lane then holds 4 neighbouring columns of one row. WV waves share a tile, two
// along m. KG groups of them take the panels in turn and add their sums up at the end: with few tiles this fills the
// CUs. Of ST panels in a group's part of LDS one is multiplied, the others are on their way.
//
// What bounds it, 2 x 4096 x 4096: P X the matrix cores under the card's power limit, 1180 TFLOP/s issued (700 us), where
// the library's fp16 product of 8192^3 reaches 1200. X X^T and A A reach 950 (445 us): their 1056 tiles on and above the
// diagonal are 4.1 a CU, and the fullest has 5. 12 x 768 x 768, 19 to 33 GFLOP issued a stage: 30 to 46 us, of which 8 to 9
// do not depend on the length of the sum, the start of a launch and the results on their way to memory behind it.
template<int KIND, int BM, int BN, int WV, int KG, int ST, DType W>
__global__ __launch_bounds__(64 * WV * KG, KG == 1 ? 2 : 4) void k_muon_product(MuonTable t, MuonStage st) {
    constexpr int WM = BM / 2, WN = BN / (WV / 2), MT = WM / 32, NT = WN / 32;
    constexpr int BK = 16; // columns of a panel, the step along the sum
    constexpr bool NN = KIND == kApply || KIND == kFinal;
    constexpr bool AHEAD = MT * NT <= 4; // registers for two tiles' fragments
    static_assert(AHEAD || KG == 1, "the other loop has no round without a panel");
    constexpr int kTile = (BM + BN) * 64;
    constexpr int kSlice = 32 * (WN + 4) * 4; // 32 rows of a wave's results, padded against bank conflicts
    constexpr int kLds = KG * (ST * kTile > WV * kSlice ? ST * kTile : WV * kSlice);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];

    const int blk = place_of_block<NN ? kBand * kBand : 32>();
    const int i = entry_of(t, blk);
    const MuonEntry &e = t.e[i];
    const int rows = e.mp;
    const int tm = (rows + BM - 1) / BM, tn = ((NN ? e.np : rows) + BN - 1) / BN;
    constexpr int R = BM / BN;
    const int b = blk - t.first[i];
    int ti, tj, which;
    if constexpr (NN) {
        which = b / (tm * tn);
        const int rest = b % (tm * tn), band = rest / (kBand * tn) * kBand, h = tm - band < kBand ? tm - band : kBand;
        ti = band + (rest - band * tn) % h;
        tj = (rest - band * tn) / h;
    } else { // tiles that reach the diagonal or lie above it
        const int tiles = tm * tn - R * (tm * (tm - 1) / 2);
        which = b / tiles;
        int rest = b % tiles;
        ti = 0;
        while (rest >= tn - R * ti) rest -= tn - R * ti++;
        tj = R * ti + rest;
    }
    const Planes q = planes_of(t.ws, e, which);
    const _Float16 *x = st.cur ? q.x1 : q.x0;
    const int m0 = ti * BM, n0 = tj * BN;
    const int K = KIND == kGram ? e.np : rows;
    const _Float16 *ms = KIND == kGram ? x : KIND == kPoly ? q.a : q.p;
    const _Float16 *ns = KIND == kPoly ? q.a : x;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % WV),
              group = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WV));
    // source of each 16-byte piece this lane brings to LDS; rows and panels past the matrix repeat its last ones
    constexpr int MI = BM / (16 * WV), NI = BN / (16 * WV);
    const _Float16 *mp[MI], *np[NI];
    const int lrow = lane >> 2;
    const int lpiece = (lane & 3) ^ swizzle(lrow);
#pragma unroll
    for (int k = 0; k < MI; ++k) {
        const int r = m0 + (wave * MI + k) * 16 + lrow;
        mp[k] = ms + (static_cast<size_t>(group) * rows + (r < rows ? r : rows - 1)) * 32 + lpiece * 8;
    }
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        if constexpr (NN) { // BK rows of BN / BK panels
            const int j = wave * NI + k, panels = e.np / BK, pn = n0 / BK + j;
            np[k] = ns + (static_cast<size_t>(pn < panels ? pn : panels - 1) * rows + group * BK + lrow) * 32 +
                    (lpiece ^ ((j & 1) << 1)) * 8;
        } else {
            const int r = n0 + (wave * NI + k) * 16 + lrow;
            np[k] = ns + (static_cast<size_t>(group) * rows + (r < rows ? r : rows - 1)) * 32 + lpiece * 8;
        }
    }
    const size_t mstep = static_cast<size_t>(rows) * 32 * KG, nstep = NN ? BK * 32 * KG : mstep;
    uint8_t *mine = lds + group * ST * kTile;
    const auto fetch = [&](int buf) {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_offset(mine + buf * kTile));
#pragma unroll
        for (int k = 0; k < MI; ++k) {
            load_to_lds(mp[k], to + (wave * MI + k) * 1024);
            mp[k] += mstep;
        }
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            load_to_lds(np[k], to + BM * 64 + (wave * NI + k) * 1024);
            np[k] += nstep;
        }
    };

    const int wm = (wave & 1) * WM, wn = (wave >> 1) * WN;
    const int half = lane >> 5, l32 = lane & 31;
    uint32_t tr[2][2] = {}; // transposed reads: 16 lanes fetch a 4 x 16 block of X and get its columns, 4 of the sum each
    if constexpr (NN) {
        const int l16 = lane & 15, cb = (lane >> 4) & 1;
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int r = 8 * half + 4 * z + (l16 >> 2);
                const int piece = 2 * s + ((l16 & 3) >> 1), panel = wn / 16 + cb;
                tr[z][s] = panel * (BK * 64) + r * 64 + ((piece ^ swizzle(r, cb)) << 4) + (l16 & 1) * 8;
            }
    }
    const _Float16 *in = NN ? x : q.a; // what the epilogue reads
    const int nmax = NN ? e.np : rows;
    constexpr int LR = WN / 8, O = 32 / (64 / LR); // lanes of a row, and pieces of a slice of 32 rows of the results
    const auto mine_of = [&](int o) { return KG == 1 || o % KG == group; }; // pieces are shared out over the groups
    const auto ask = [&](int u, half8 (&ih)[O], half8 (&il)[O]) {
#pragma unroll
        for (int o = 0; o < O; ++o) {
            const int m = m0 + wm + u * 32 + o * (64 / LR) + lane / LR, n = n0 + wn + lane % LR * 8;
            if (mine_of(o) && m < rows && n < nmax) {
                const size_t at = panel_at(rows, m, n);
                ih[o] = *reinterpret_cast<const half8 *>(in + at);
                il[o] = *reinterpret_cast<const half8 *>(in + at + kLo);
            }
        }
    };
    constexpr bool kAskFirst = KIND != kGram && KG > 1; // few tiles: nothing else would hide these loads
    half8 eh[kAskFirst ? MT : 1][O], el[kAskFirst ? MT : 1][O];
    if constexpr (kAskFirst) {
#pragma unroll
        for (int u = 0; u < MT; ++u) ask(u, eh[u], el[u]);
    }
    float16v acc[NT][MT] = {};
    const int panels = K / BK, rounds = (panels + KG - 1) / KG, steps = (panels - group + KG - 1) / KG; // this group's
    const auto read = [&](int buf, half8 (&mf)[MT][2], half8 (&nf)[NT][2]) {
        // [0]: the hi parts of 16 of the sum, [1]: the lo parts
        const uint8_t *ml = mine + buf * kTile, *nl = ml + BM * 64;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int at = l32 * 64 + (((2 * s + half) ^ swizzle(l32)) << 4);
#pragma unroll
            for (int u = 0; u < MT; ++u) mf[u][s] = *reinterpret_cast<const half8 *>(ml + (wm + u * 32) * 64 + at);
            if constexpr (!NN) {
#pragma unroll
                for (int y = 0; y < NT; ++y) nf[y][s] = *reinterpret_cast<const half8 *>(nl + (wn + y * 32) * 64 + at);
            }
        }
        if constexpr (NN) read_transposed<NT, 32 * 64>(nl, tr, nf);
    };
    const auto multiply = [&](const half8 (&mf)[MT][2], const half8 (&nf)[NT][2]) {
        const auto mul = [&](int sn, int sm) {
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
                for (int u = 0; u < MT; ++u)
                    acc[y][u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(nf[y][sn], mf[u][sm], acc[y][u], 0, 0, 0);
        };
        mul(0, 0);
        mul(0, 1);
        mul(1, 0);
    };
    if constexpr (AHEAD) {
        // the next tile's fragments are read while this one's are multiplied
        half8 mf[2][MT][2], nf[2][NT][2];
#pragma unroll
        for (int k = 0; k < ST; ++k)
            if (k < steps) fetch(k);
        wait_tiles<MI + NI, ST>(steps - 1 < ST - 1 ? (steps > 1 ? steps - 1 : 0) : ST - 1);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (steps > 0) read(0, mf[0], nf[0]);
        int buf = 0;
        const auto round = [&](int k, int set) {
            const int next = buf == ST - 1 ? 0 : buf + 1, later = steps - 2 - k; // tiles behind the next one
            wait_tiles<MI + NI, ST - 1>(later < ST - 2 ? (later > 0 ? later : 0) : ST - 2);
            __builtin_amdgcn_s_barrier(); // tile k + 1 has landed for every wave, and all have read tile k
            asm volatile("" ::: "memory");
            if (k + 1 < steps) read(next, mf[set ^ 1], nf[set ^ 1]);
            if (k + ST < steps) fetch(buf);
            if (k < steps) multiply(mf[set], nf[set]);
            buf = next;
        };
        for (int k = 0; k < rounds; k += 2) {
            round(k, 0);
            if (k + 1 < rounds) round(k + 1, 1);
        }
    } else {
#pragma unroll
        for (int k = 0; k < ST - 1; ++k)
            if (k < steps) fetch(k);
        for (int k = 0, buf = 0, to = ST - 1; k < steps; ++k) {
            const int later = steps - 1 - k; // tiles behind this one
            wait_tiles<MI + NI, ST - 1>(later < ST - 2 ? (later > 0 ? later : 0) : ST - 2);
            __builtin_amdgcn_s_barrier(); // tile k has landed for every wave, and all are done with tile k - 1
            asm volatile("" ::: "memory");
            half8 mf[MT][2], nf[NT][2];
            read(buf, mf, nf);
            if (k + ST - 1 < steps) fetch(to); // over tile k - 1
            buf = buf == ST - 1 ? 0 : buf + 1;
            to = to == ST - 1 ? 0 : to + 1;
            multiply(mf, nf);
        }
    }
    __syncthreads(); // the tiles' memory now carries results

    // Results leave through LDS, 32 rows of a wave at a time: a lane then has 8 neighbouring columns of a row. What it
    // needs from memory is asked for before. Of a symmetric result only the 32 x 32 blocks on and above the diagonal are
    // used: hi lo + lo hi is not lo hi + hi lo in floating point, and the mirrored half comes from the other.
    const bool flip = e.rows > e.cols;
    const int small = flip ? e.cols : e.rows, large = flip ? e.rows : e.cols;
    constexpr int kPitch = WN + 4;
    // a wave's slice of its own sums, the first group's (the whole sum's), and what orders accesses to them
    float *own = reinterpret_cast<float *>(lds + (group * WV + wave) * kSlice);
    float *slice = reinterpret_cast<float *>(lds + wave * kSlice);
    const auto sync = [] {
        if constexpr (KG == 1)
            wave_sync();
        else
            __syncthreads();
    };
    using WS = typename Elem<W>::S;
    WS *w = KIND == kFinal ? static_cast<WS *>(e.w) + static_cast<size_t>(e.rows) * e.cols * which : nullptr;
    const float alpha = e.alpha;
    const bool step = e.mom != nullptr;
    const auto final_value = [&](float v, WS old) {
        v *= 1.0f / kMuonScaleX;
        return static_cast<WS>(step ? static_cast<float>(old) * st.decay - alpha * v : v);
    };
    _Float16 *out = KIND == kGram ? q.a : KIND == kPoly ? q.p : st.cur ? q.x0 : q.x1;
#pragma unroll
    for (int u = 0; u < MT; ++u) {
        const int mb = m0 + wm + u * 32;
        half8 ih[O], il[O];
        if constexpr (kAskFirst) {
#pragma unroll
            for (int o = 0; o < O; ++o) {
                ih[o] = eh[u][o];
                il[o] = el[u][o];
            }
        } else if constexpr (KIND != kGram) {
            ask(u, ih, il);
        }
#pragma unroll
        for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float4 v;
                v.x = acc[y][u][4 * k];
                v.y = acc[y][u][4 * k + 1];
                v.z = acc[y][u][4 * k + 2];
                v.w = acc[y][u][4 * k + 3];
                *reinterpret_cast<float4 *>(own + l32 * kPitch + y * 32 + 8 * k + 4 * half) = v;
            }
        sync();
#pragma unroll
        for (int o = 0; o < O; ++o) {
            const int r = o * (64 / LR) + lane / LR, c = lane % LR * 8;
            const int m = mb + r, n = n0 + wn + c;
            if (!mine_of(o) || m >= rows || n >= nmax || (!NN && (n | 31) < mb)) continue;
            float v[8];
            *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(slice + r * kPitch + c);
            *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(slice + r * kPitch + c + 4);
#pragma unroll
            for (int j = 1; j < KG; ++j) {
                const float *other = slice + j * WV * (kSlice / 4) + r * kPitch + c;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] += other[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (KIND == kGram) {
                    v[k] *= kMuonScaleA / (kMuonScaleX * kMuonScaleX);
                } else {
                    const float old = join_fp16(ih[o][k], il[o][k]);
                    if constexpr (NN)
                        v[k] = __builtin_fmaf(st.a, old, v[k] * (1.0f / kMuonScaleP));
                    else
                        v[k] = __builtin_fmaf(st.b * (kMuonScaleP / kMuonScaleA), old,
                                              v[k] * (st.c * (kMuonScaleP / (kMuonScaleA * kMuonScaleA))));
                }
            }
            if constexpr (KIND != kFinal) {
                half8 oh, ol;
                split_fp16<8>(v, oh, ol);
                const size_t at = panel_at(rows, m, n);
                *reinterpret_cast<half8 *>(out + at) = oh;
                *reinterpret_cast<half8 *>(out + at + kLo) = ol;
            }
            if (KIND != kApply) { // read again, along the columns or by other lanes
                *reinterpret_cast<float4 *>(slice + r * kPitch + c) = *reinterpret_cast<float4 *>(v);
                *reinterpret_cast<float4 *>(slice + r * kPitch + c + 4) = *reinterpret_cast<float4 *>(v + 4);
            }
        }
        sync();
        if constexpr (!NN) {
            // the mirrored half: 8 of the 32 rows of one column per lane
            if (n0 + wn + WN > mb + 32 && mb < rows) {
#pragma unroll
                for (int o = 0; o < WN; o += 16) {
                    const int c = o + (lane >> 2), r = (lane & 3) * 8;
                    const int n = n0 + wn + c;
                    if (!mine_of(o / 16) || n >= rows || n < mb + 32) continue;
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = slice[(r + k) * kPitch + c];
                    half8 oh, ol;
                    split_fp16<8>(v, oh, ol);
                    const size_t at = panel_at(rows, n, mb + r);
                    *reinterpret_cast<half8 *>(out + at) = oh;
                    *reinterpret_cast<half8 *>(out + at + kLo) = ol;
                }
            }
        }
        if constexpr (KIND == kFinal) {
            // the caller's matrix: its rows lie along n, or along m where it was transposed; 4 elements per lane
            constexpr int P = WN * 32 / 256; // pieces of a slice
            const int lr = flip ? lane >> 3 : lane / (WN / 4), lc = flip ? (lane & 7) * 4 : lane % (WN / 4) * 4;
            Run<WS, 4> old[P];
            bool whole[P];
            size_t at[P];
#pragma unroll
            for (int k = 0; k < P; ++k) { // rows of the caller's: n = lr + 8 k, or m = lr + (256 / WN) k
                const int m = flip ? mb + lc : mb + lr + 256 / WN * k;
                const int n = flip ? n0 + wn + lr + 8 * k : n0 + wn + lc;
                at[k] = flip ? static_cast<size_t>(n) * e.cols + m : static_cast<size_t>(m) * e.cols + n;
                whole[k] = flip ? n < large && m + 4 <= small : m < small && n + 4 <= large;
                if (mine_of(k) && whole[k] && step) old[k] = *reinterpret_cast<const Run<WS, 4> *>(w + at[k]);
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                if (!mine_of(k)) continue;
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[j] = flip ? slice[(lc + j) * kPitch + lr + 8 * k] : slice[(lr + 256 / WN * k) * kPitch + lc + j];
                if (whole[k]) {
                    Run<WS, 4> now;
#pragma unroll
                    for (int j = 0; j < 4; ++j) now.v[j] = final_value(v[j], old[k].v[j]);
                    *reinterpret_cast<Run<WS, 4> *>(w + at[k]) = now;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int m = flip ? mb + lc + j : mb + lr + 256 / WN * k;
                        const int n = flip ? n0 + wn + lr + 8 * k : n0 + wn + lc + j;
                        if (m < small && n < large) w[at[k] + j] = final_value(v[j], step ? w[at[k] + j] : WS{});
                    }
                }
            }
        }
        sync();
    }
}

// Everything for a matrix that fits in LDS, by one workgroup: X, and A / P in one place, in paired panels as above and
// with three products, up to 32 rows four for A and A A. A wave has whole 32 x 32 tiles of the products, so nothing is joined between waves,
// and keeps its own entries of X and A in registers from product to product. Bound by LDS reads, products and barriers
// in turn; us of a call of orthogonalize / the Muon step: 64 x 64 14 / 16 (4 waves; sharing each tile's sum between 2
// or 4 waves 17 / 21), 64 x 256 28 / 31 (8 waves; 4, which read least, 36), 256 x 64 29 / 32, 128 x 128 39 / 42 (16
// waves; 8 40 / 43). 1000 of 64 x 64 40 us. The 17 launches of the stages took 77 for 64 x 64.
template<int MP, int NP, int NW, DType G, DType W>
__global__ __launch_bounds__(64 * NW) void k_muon_small(MuonTable t, MuonParams p) {
    using S = typename Elem<G>::S;
    using WS = typename Elem<W>::S;
    constexpr int MB = MP / 32;
    constexpr int NA = NW < MB * MB ? NW : MB * MB; // waves that have tiles of A
    constexpr int RA = MB * MB / NA;                // tiles of A of such a wave, one under the other
    constexpr int RM = MB * (NP / 32) / NW;         // tiles of X of a wave, one under the other
    constexpr int E = MP * NP / (512 * NW);         // groups of 8 elements per thread
    static_assert((MP == 64 || MP == 128) && RA * NA == MB * MB && RM * NW == MB * (NP / 32) && MB % RM == 0);
    __shared__ __attribute__((aligned(16))) uint8_t lx[MP * NP * 4];
    __shared__ __attribute__((aligned(16))) uint8_t la[MP * MP * 4];
    __shared__ double sums[NW];

    const int i = entry_of(t, blockIdx.x);
    const MuonEntry &e = t.e[i];
    const int which = blockIdx.x - t.first[i];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5, l32 = lane & 31;
    const size_t elems = static_cast<size_t>(e.rows) * e.cols * which;
    const S *g = static_cast<const S *>(e.g) + elems;
    WS *w = static_cast<WS *>(e.w) + elems;
    float *mom = e.mom ? e.mom + elems : nullptr;
    const bool flip = e.rows > e.cols;
    const int np = e.np;

    const int ms = flip ? e.cols : e.rows, ns = flip ? e.rows : e.cols;
    const auto place = [&](int m, int n) { return flip ? n * e.cols + m : m * e.cols + n; };

    // Momentum, and the norm; the update stays in registers, 8 neighbouring columns of a row of X per group. The lanes
    // of a wave lie along the caller's rows: 8 x 8 groups, or 64 rows where X is the transpose.
    float u[E][8];
    int gm[E], gn[E];
    bool whole[E], tall[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int unit = threadIdx.x + 64 * NW * k, in = unit & 63, blk = unit >> 6;
        gm[k] = flip ? blk % (MP / 64) * 64 + in : blk % (MP / 8) * 8 + (in >> 3);
        gn[k] = flip ? blk / (MP / 64) * 8 : (blk / (MP / 8) * 8 + (in & 7)) * 8;
        whole[k] = !flip && gm[k] < ms && gn[k] + 8 <= ns; // 8 neighbours in the caller's memory too
        tall[k] = flip && gm[k] < ms && gn[k] + 8 <= ns;   // 8 loads or stores without a condition each
        if (whole[k]) {
            const Run<S, 8> v = *reinterpret_cast<const Run<S, 8> *>(g + place(gm[k], gn[k]));
#pragma unroll
            for (int j = 0; j < 8; ++j) u[k][j] = static_cast<float>(v.v[j]);
        } else if (tall[k]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[k][j] = static_cast<float>(g[place(gm[k], gn[k] + j)]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                u[k][j] = gm[k] < ms && gn[k] + j < ns ? static_cast<float>(g[place(gm[k], gn[k] + j)]) : 0.0f;
        }
    }
    if (mom) {
        Run<float, 8> old[E];
#pragma unroll
        for (int k = 0; k < E; ++k) {
            if (whole[k]) {
                old[k] = *reinterpret_cast<const Run<float, 8> *>(mom + place(gm[k], gn[k]));
            } else if (tall[k]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) old[k].v[j] = mom[place(gm[k], gn[k] + j)];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    old[k].v[j] = gm[k] < ms && gn[k] + j < ns ? mom[place(gm[k], gn[k] + j)] : 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < E; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float now = old[k].v[j] + (1.0f - p.momentum) * (u[k][j] - old[k].v[j]);
                old[k].v[j] = now;
                u[k][j] = update_of(u[k][j], now, p);
            }
            if (whole[k]) {
                *reinterpret_cast<Run<float, 8> *>(mom + place(gm[k], gn[k])) = old[k];
            } else if (tall[k]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) mom[place(gm[k], gn[k] + j)] = old[k].v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (gm[k] < ms && gn[k] + j < ns) mom[place(gm[k], gn[k] + j)] = old[k].v[j];
            }
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < E; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += static_cast<double>(u[k][j]) * u[k][j];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < NW; ++k) sum += sums[k];
    const double norm = sqrt(sum);
    const double scale = static_cast<double>(kMuonScaleX) / (norm > p.eps || norm != norm ? norm : p.eps);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        if (gm[k] >= MP || gn[k] >= np) continue; // more groups than elements
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(u[k][j] * scale);
        half8 h, l;
        split_fp16<8>(v, h, l);
        uint8_t *row = lx + ((gn[k] >> 4) * MP + gm[k]) * 64;
        const int at = ((gn[k] >> 3) & 1) ^ swizzle(gm[k], gn[k] >> 4);
        *reinterpret_cast<half8 *>(row + (at << 4)) = h;
        *reinterpret_cast<half8 *>(row + ((at ^ 2) << 4)) = l;
    }

    // What a lane adds to a tile's place: fragments of 32 rows along the sum, fragments through the transposing read,
    // and its 4 columns of a row of a result ([lo][second 8 columns of a panel][odd panel]).
    const int sw = swizzle(l32);
    int fo[2], to[2][2], ro[2][2][2];
#pragma unroll
    for (int lo = 0; lo < 2; ++lo) {
        fo[lo] = l32 * 64 + (((2 * lo + half) ^ sw) << 4);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int l16 = lane & 15, cb = (lane >> 4) & 1, r = 8 * half + 4 * z + (l16 >> 2);
            to[z][lo] = (cb * MP + r) * 64 + (((2 * lo + ((l16 & 3) >> 1)) ^ swizzle(r, cb)) << 4) + (l16 & 1) * 8;
#pragma unroll
            for (int odd = 0; odd < 2; ++odd)
                ro[lo][z][odd] = l32 * 64 + (((2 * lo + z) ^ sw ^ (odd << 1)) << 4) + 8 * half;
        }
    }
    const auto frag = [&](const uint8_t *base, int r0, int panel, int lo) {
        return *reinterpret_cast<const half8 *>(base + (panel * MP + r0) * 64 + (panel & 1 ? fo[lo] ^ 32 : fo[lo]));
    };
    const auto frag_t = [&](const uint8_t *base, int k0, int n0, int lo) {
        half4 h[2];
#pragma unroll
        for (int z = 0; z < 2; ++z)
            h[z] = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                 (__attribute__((address_space(3))) short4v *)(
                                                     base + (n0 / 16 * MP + k0) * 64 + to[z][lo])));
        return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
    };
    const auto mul3 = [](float16v c, const half8 (&n)[2], const half8 (&m)[2]) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(n[0], m[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(n[0], m[1], c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(n[1], m[0], c, 0, 0, 0);
    };
    // group b of 4 columns: a result's byte without the lane's part
    const auto group_at = [&](int mt, int nt, int b) { return ((nt / 16 + (b >> 1)) * MP + mt) * 64; };
    const auto put4 = [&](uint8_t *base, int at, int b, const float (&v)[4]) {
        half4 oh, ol;
        split_fp16<4>(v, oh, ol);
        *reinterpret_cast<half4 *>(base + at + ro[0][b & 1][b >> 1]) = oh;
        *reinterpret_cast<half4 *>(base + at + ro[1][b & 1][b >> 1]) = ol;
    };
    const auto get4 = [&](const uint8_t *base, int at, int b, float (&v)[4]) {
        const half4 h = *reinterpret_cast<const half4 *>(base + at + ro[0][b & 1][b >> 1]);
        const half4 l = *reinterpret_cast<const half4 *>(base + at + ro[1][b & 1][b >> 1]);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = join_fp16(h[r], l[r]);
    };
    // where this wave's tiles lie: of A in rows ar + 32 k, of X in rows xr + 32 k
    const int ar = wave * RA % MB * 32, ac = wave * RA / MB * 32;
    const int xr = wave * RM % MB * 32, xc = wave * RM / MB * 32;
    const bool has_a = NA == NW || wave < NA, has_x = NP == MP || xc < np;
    // This wave's tiles of `base` times its own transpose. hi lo + lo hi get a sum of their own (in one sum with hi hi they
    // round it three times as often), and up to 32 rows lo lo is added too: so few rows leave nothing for these roundings to
    // average out over. Error over that of the same steps in fp32, 64 x 64 0.88 -> 0.76 (14.0 -> 14.4 us), 64 x 256 1.0 -> 0.8
    // (26.8 -> 27.9), 16 x 230 1.8 -> 1.3 (27.4 -> 29.7; without lo lo 1.45); 128 x 128 0.8 as it is, with no register free.
    constexpr bool kApart = MP == 64;
    const auto square_by = [&](auto four, const uint8_t *base, int panels, float16v (&out)[RA]) {
        float16v low[kApart ? RA : 1] = {};
#pragma unroll
        for (int k = 0; k < RA; ++k) out[k] = float16v{};
#pragma unroll (MP == 128 ? 2 : 4)
        for (int s = 0; s < panels; ++s) {
            const half8 n[2] = {frag(base, ac, s, 0), frag(base, ac, s, 1)};
#pragma unroll
            for (int k = 0; k < RA; ++k) {
                const half8 m[2] = {frag(base, ar + 32 * k, s, 0), frag(base, ar + 32 * k, s, 1)};
                if constexpr (kApart) {
                    out[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(n[0], m[0], out[k], 0, 0, 0);
                    low[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(n[0], m[1], low[k], 0, 0, 0);
                    low[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(n[1], m[0], low[k], 0, 0, 0);
                    if constexpr (decltype(four)::value)
                        low[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(n[1], m[1], low[k], 0, 0, 0);
                } else {
                    out[k] = mul3(out[k], n, m);
                }
            }
        }
        if constexpr (kApart) {
#pragma unroll
            for (int k = 0; k < RA; ++k) out[k] += low[k];
        }
    };
    const auto square = [&](const uint8_t *base, int panels, float16v (&out)[RA]) {
        if (kApart && ms <= 32)
            square_by(std::true_type{}, base, panels, out);
        else
            square_by(std::false_type{}, base, panels, out);
    };

    __syncthreads(); // X is written
    float x[RM][16]; // this wave's entries of X
    if (has_x)
#pragma unroll
        for (int k = 0; k < RM; ++k)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float v[4];
                get4(lx, group_at(xr + 32 * k, xc, b), b, v);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[k][4 * b + r] = v[r];
            }
    for (int step = 0; step < p.steps; ++step) {
        float16v sq[RA], aa[RA];
        if (has_a) {
            square(lx, NP == MP ? MP / 16 : np / 16, sq);
#pragma unroll
            for (int k = 0; k < RA; ++k)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = sq[k][4 * b + r] *= kMuonScaleA / (kMuonScaleX * kMuonScaleX);
                    put4(la, group_at(ar + 32 * k, ac, b), b, v);
                }
        }
        __syncthreads(); // A is written
        if (has_a) square(la, MP / 16, aa);
        __syncthreads(); // A is read; P takes its place
        if (has_a)
#pragma unroll
            for (int k = 0; k < RA; ++k)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        v[r] = __builtin_fmaf(p.b * (kMuonScaleP / kMuonScaleA), sq[k][4 * b + r],
                                              aa[k][4 * b + r] * (p.c * (kMuonScaleP / (kMuonScaleA * kMuonScaleA))));
                    put4(la, group_at(ar + 32 * k, ac, b), b, v);
                }
        __syncthreads(); // P is written
        const bool last = step == p.steps - 1;
        Run<WS, 4> old[RM][4];
        float16v px[RM] = {};
        if (has_x) {
            if (last && mom) { // on their way while P X is computed
#pragma unroll
                for (int k = 0; k < RM; ++k)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int m = xr + 32 * k + l32, n = xc + 4 * half + 8 * b;
                        if (!flip && m < ms && n + 4 <= ns) {
                            old[k][b] = *reinterpret_cast<const Run<WS, 4> *>(w + place(m, n));
                        } else if (m < ms && n + 4 <= ns) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) old[k][b].v[r] = w[place(m, n + r)];
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                old[k][b].v[r] = m < ms && n + r < ns ? w[place(m, n + r)] : WS{};
                        }
                    }
            }
#pragma unroll
            for (int s = 0; s < MP / 16; ++s) {
                const half8 n[2] = {frag_t(lx, 16 * s, xc, 0), frag_t(lx, 16 * s, xc, 1)};
#pragma unroll
                for (int k = 0; k < RM; ++k) {
                    const half8 m[2] = {frag(la, xr + 32 * k, s, 0), frag(la, xr + 32 * k, s, 1)};
                    px[k] = mul3(px[k], n, m);
                }
            }
        }
        __syncthreads(); // X is read
        if (has_x)
#pragma unroll
            for (int k = 0; k < RM; ++k)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        v[r] = x[k][4 * b + r] =
                            __builtin_fmaf(p.a, x[k][4 * b + r], px[k][4 * b + r] * (1.0f / kMuonScaleP));
                    if (!last) {
                        put4(lx, group_at(xr + 32 * k, xc, b), b, v);
                        continue;
                    }
                    const int m = xr + 32 * k + l32, n = xc + 4 * half + 8 * b;
                    Run<WS, 4> now;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float o = v[r] * (1.0f / kMuonScaleX);
                        now.v[r] =
                            static_cast<WS>(mom ? static_cast<float>(old[k][b].v[r]) * p.decay - e.alpha * o : o);
                    }
                    if (!flip && m < ms && n + 4 <= ns) {
                        *reinterpret_cast<Run<WS, 4> *>(w + place(m, n)) = now;
                    } else if (m < ms && n + 4 <= ns) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) w[place(m, n + r)] = now.v[r];
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m < ms && n + r < ns) w[place(m, n + r)] = now.v[r];
                    }
                }
        if (!last) __syncthreads(); // X is written
    }
}

namespace {

// fills in the first workgroup of every entry; returns their number
template<typename F>
int64_t layout(MuonTable &t, F &&blocks) {
    int64_t n = 0;
    for (int i = 0; i < t.n; ++i) {
        t.first[i] = static_cast<int>(n);
        n += static_cast<int64_t>(blocks(t.e[i])) * t.e[i].count;
    }
    return n;
}

// tiles of one matrix in a product stage
template<int BM, int BN>
int64_t product_tiles(int kind, const MuonEntry &e) {
    const int64_t tm = (e.mp + BM - 1) / BM;
    if (kind == kApply || kind == kFinal) return tm * ((e.np + BN - 1) / BN);
    return tm * ((e.mp + BN - 1) / BN) - BM / BN * (tm * (tm - 1) / 2);
}

template<int KIND, int BM, int BN, int WV, int KG, int ST, DType W>
bool launch_product(MuonTable &t, const MuonStage &st, hipStream_t s) {
    const int64_t n = layout(t, [](const MuonEntry &e) { return product_tiles<BM, BN>(KIND, e); });
    if (n > INT32_MAX) return false;
    const dim3 grid(static_cast<unsigned>(n));
    return launch_ok([&] { k_muon_product<KIND, BM, BN, WV, KG, ST, W><<<grid, 64 * WV * KG, 0, s>>>(t, st); });
}

template<int KIND, DType W = DType::F32>
bool launch_stage(MuonTable &t, const MuonStage &st, hipStream_t s) {
    // Tiles by an estimate of a launch's time: some us, and for each panel of the sum the time of a tile times the tiles
    // of a CU, between the average and the fullest CU's (where two fit a CU an odd one out takes a quarter longer, where
    // one fits the fullest counts). Fitted to 44 calls in two types; the tiles chosen cost 1 % over the best of each launch
    // on average. In us, fp32, X X^T / P X, for 256 x 128, 128 x 128, 128 x 64, 64 x 64 by two groups of waves and by
    // four, 64 x 32 by four:
    //   1 x 512 x 512       27 / 29     17 / 19     13 / 14      9 / 10      9 / 9       7 / 7
    //   1 x 1024 x 1024     44 / 47     29 / 31     21 / 23     14 / 16     13 / 14     13 / 14
    //   12 x 768 x 768      41 / 46     30 / 40     29 / 46     30 / 54     39 / 70     38 / 64
    //   4 x 1024 x 4096    157 / 102   105 / 107    94 / 116    88 / 155   100 / 190   101 / 188
    //   2 x 4096 x 4096    493 / 680   438 / 740   473 / 846   609 / 1023  658 / 1172  669 / 1254
    double panels = 0.0, all = 0.0;
    for (int i = 0; i < t.n; ++i) {
        const double tiles = static_cast<double>(t.e[i].count) * product_tiles<64, 64>(KIND, t.e[i]);
        panels += tiles * (KIND == kGram ? t.e[i].np : t.e[i].mp) / 16;
        all += tiles;
    }
    panels /= all;
    const auto cost = [&](auto tiles_of, double launch, double tile, bool two_fit = true) {
        int64_t tiles = 0;
        for (int i = 0; i < t.n; ++i) tiles += t.e[i].count * tiles_of(t.e[i]);
        const int64_t fullest = (tiles + 255) / 256;
        const double average = std::max(tiles / 256.0, 1.0);
        return launch + panels * tile * (two_fit ? 0.5 * (average + fullest) + (fullest & 1) * 0.26 : fullest);
    };
    const double est[6] = {
        cost([](const MuonEntry &e) { return product_tiles<256, 128>(KIND, e); }, 6.0, 0.600),
        cost([](const MuonEntry &e) { return product_tiles<128, 128>(KIND, e); }, 6.9, 0.313),
        cost([](const MuonEntry &e) { return product_tiles<128, 64>(KIND, e); }, 4.5, 0.207),
        cost([](const MuonEntry &e) { return product_tiles<64, 64>(KIND, e); }, 4.2, 0.125),
        cost([](const MuonEntry &e) { return product_tiles<64, 64>(KIND, e); }, 4.4, 0.149, false),
        cost([](const MuonEntry &e) { return product_tiles<64, 32>(KIND, e); }, 4.2, 0.084),
    };
    switch (std::min_element(est, est + 6) - est) {
        case 0: return launch_product<KIND, 256, 128, 4, 1, 3, W>(t, st, s);
        case 1: return launch_product<KIND, 128, 128, 4, 1, 3, W>(t, st, s);
        case 2: return launch_product<KIND, 128, 64, 4, 1, 3, W>(t, st, s);
        case 3: return launch_product<KIND, 64, 64, 4, 2, 3, W>(t, st, s);
        case 4: return launch_product<KIND, 64, 64, 4, 4, 3, W>(t, st, s);
        default: return launch_product<KIND, 64, 32, 2, 4, 3, W>(t, st, s);
    }
}

} // namespace

template<int MP, int NP, int NW, DType G>
static bool launch_small(MuonTable &t, DType wt, const MuonParams &p, hipStream_t s) {
    const int64_t n = layout(t, [](const MuonEntry &) { return 1; });
    if (n > INT32_MAX) return false;
    const dim3 grid(static_cast<unsigned>(n));
    return launch_ok([&] {
        if (wt == DType::F32)
            k_muon_small<MP, NP, NW, G, DType::F32><<<grid, 64 * NW, 0, s>>>(t, p);
        else if (wt == DType::BF16)
            k_muon_small<MP, NP, NW, G, DType::BF16><<<grid, 64 * NW, 0, s>>>(t, p);
        else
            k_muon_small<MP, NP, NW, G, DType::F16><<<grid, 64 * NW, 0, s>>>(t, p);
    });
}

bool launch_muon(const MuonEntry *entries, int n, DType gt, DType wt, const MuonParams &p, void *ws, hipStream_t s) {
    MuonTable t{}, narrow{}, square{}; // of the stages, and of one workgroup a matrix
    t.ws = static_cast<uint8_t *>(ws);
    int np = 0;
    for (int i = 0; i < n; ++i) {
        MuonTable &to = !kernels::muon_fits_lds(entries[i].mp, entries[i].np) ? t : entries[i].mp == 64 ? narrow : square;
        to.e[to.n++] = entries[i];
        if (&to == &narrow) np = np > entries[i].np ? np : entries[i].np;
    }
    const auto with_grad = [&](auto &&f) {
        switch (gt) {
            case DType::F32: return f(std::integral_constant<DType, DType::F32>{});
            case DType::BF16: return f(std::integral_constant<DType, DType::BF16>{});
            case DType::F16: return f(std::integral_constant<DType, DType::F16>{});
            default: return false;
        }
    };
    const bool started = with_grad([&](auto g) {
        constexpr DType G = decltype(g)::value;
        if (square.n && !launch_small<128, 128, 16, G>(square, wt, p, s)) return false;
        if (narrow.n && !(np > 64 ? launch_small<64, 256, 8, G>(narrow, wt, p, s)
                                  : launch_small<64, 64, 4, G>(narrow, wt, p, s)))
            return false;
        if (t.n == 0) return true;
        int64_t blocks = layout(t, [](const MuonEntry &e) { return e.partials; });
        if (blocks > INT32_MAX) return false;
        if (!launch_ok([&] { k_muon_momentum<G><<<dim3(static_cast<unsigned>(blocks)), 256, 0, s>>>(t, p); }))
            return false;
        blocks = layout(t, [](const MuonEntry &e) { return static_cast<int64_t>(e.mp / 64) * (e.np / 64); });
        if (blocks > INT32_MAX) return false;
        return launch_ok([&] { k_muon_start<G><<<dim3(static_cast<unsigned>(blocks)), 256, 0, s>>>(t, p); });
    });
    if (!started) return false;
    if (t.n == 0) return true;
    // the longest sums first, so that the launch does not end with one: by n for X X^T, by m for the others
    MuonTable by_n = t;
    std::stable_sort(t.e, t.e + t.n, [](const MuonEntry &x, const MuonEntry &y) { return x.mp > y.mp; });
    std::stable_sort(by_n.e, by_n.e + by_n.n, [](const MuonEntry &x, const MuonEntry &y) { return x.np > y.np; });
    for (int k = 0; k < p.steps; ++k) {
        const MuonStage st{k & 1, p.a, p.b, p.c, p.decay};
        bool ok = launch_stage<kGram>(by_n, st, s) && launch_stage<kPoly>(t, st, s);
        if (!ok) return false;
        if (k + 1 < p.steps)
            ok = launch_stage<kApply>(t, st, s);
        else if (wt == DType::F32)
            ok = launch_stage<kFinal, DType::F32>(t, st, s);
        else if (wt == DType::F16)
            ok = launch_stage<kFinal, DType::F16>(t, st, s);
        else
            ok = launch_stage<kFinal, DType::BF16>(t, st, s);
        if (!ok) return false;
    }
    return true;
}

} // namespace pccl::hipk
