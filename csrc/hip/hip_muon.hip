// Newton-Schulz orthogonalisation and the Muon step (formulas, number formats and plan: csrc/kernels/muon_common.hpp).
//
// All matrices of a call, of whatever shapes, go through each stage in one launch: a workgroup finds its matrix and
// tile from its index. Stages: momentum and sums of squares; X_0 in two fp16 parts, padded, on its shorter side; then
// per step A = X X^T and P = b A + c A A over the tiles on and above the diagonal (both halves are written), and
// a X + P X, whose last pass updates the caller's parameters instead of writing X. No atomics and a fixed order of
// every sum: equal calls give equal bits, which the peers of a run rely on.
//
// The products of the 16-bit types: where the result is bf16 (8 bits), A and P X use the hi parts alone (11 bits) and
// only A A, the cheapest, all three; the term a X always has both parts, so small singular values, which the steps
// amplify up to a^steps, keep their precision. Other results use three products everywhere, the error of fp32 products.
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
    const int lane = threadIdx.x & 63;
    const bool before = lane < t.n && t.first[lane < t.n ? lane : 0] <= b;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
}

struct Planes { // one matrix in the workspace
    _Float16 *x0, *x1, *a, *p;
    double *part;
    size_t xs, as; // hi -> lo distance
};
__device__ __forceinline__ Planes planes_of(uint8_t *ws, const MuonEntry &e, int which) {
    Planes q;
    q.xs = static_cast<size_t>(e.mp) * e.np;
    q.as = static_cast<size_t>(e.mp) * e.mp;
    const size_t bytes = 2 * (4 * q.xs + 4 * q.as) + kMuonMaxPartials * sizeof(double);
    uint8_t *base = ws + e.off + bytes * which;
    q.x0 = reinterpret_cast<_Float16 *>(base);
    q.x1 = q.x0 + 2 * q.xs;
    q.a = q.x1 + 2 * q.xs;
    q.p = q.a + 2 * q.as;
    q.part = reinterpret_cast<double *>(q.p + 2 * q.as);
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

__device__ __forceinline__ float load_as(const void *p, size_t i, DType t) {
    if (t == DType::F32) return static_cast<const float *>(p)[i];
    if (t == DType::BF16) return static_cast<float>(static_cast<const __bf16 *>(p)[i]);
    return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
}
__device__ __forceinline__ void store_as(void *p, size_t i, DType t, float v) {
    if (t == DType::F32)
        static_cast<float *>(p)[i] = v;
    else if (t == DType::BF16)
        static_cast<__bf16 *>(p)[i] = static_cast<__bf16>(v);
    else
        static_cast<_Float16 *>(p)[i] = static_cast<_Float16>(v);
}

// sum over a workgroup of 256 in a fixed order, the same in every thread
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double w[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
    __syncthreads();
    return (w[0] + w[1]) + (w[2] + w[3]);
}

__device__ __forceinline__ float update_of(float g, float m, const MuonParams &p) {
    return p.nesterov ? g + p.momentum * (m - g) : m;
}

} // namespace

// B += (1 - mu)(G - B), and the squares of U summed in 64 bits (a gradient's squares leave fp32's range long before
// the gradient does). Memory bound.
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
    for (size_t k = s0 + threadIdx.x; k < s1; k += 256) {
        float u = static_cast<float>(g[k]);
        if (m) {
            const float old = m[k];
            const float now = old + (1.0f - p.momentum) * (u - old);
            m[k] = now;
            u = update_of(u, now, p);
        }
        sum += static_cast<double>(u) * u;
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) planes_of(t.ws, e, which).part[part] = sum;
}

// X_0 = U scale / max(||U||, eps) in two fp16 parts, 64 x 64 tiles; a tall U is transposed through LDS.
template<DType G>
__global__ __launch_bounds__(256) void k_muon_start(MuonTable t, MuonParams p) {
    using S = typename Elem<G>::S;
    __shared__ float tile[64][65];
    const int i = entry_of(t, blockIdx.x);
    const MuonEntry &e = t.e[i];
    const int tn = e.np / 64, tiles = e.mp / 64 * tn;
    const int b = blockIdx.x - t.first[i], which = b / tiles, m0 = b % tiles / tn * 64, n0 = b % tiles % tn * 64;
    const Planes q = planes_of(t.ws, e, which);
    double sum = 0.0;
    for (int k = threadIdx.x; k < e.partials; k += 256) sum += q.part[k];
    sum = block_sum(sum);
    const double norm = sqrt(sum);
    const double scale = static_cast<double>(kMuonScaleX) / (norm > p.eps || norm != norm ? norm : p.eps);
    const size_t elems = static_cast<size_t>(e.rows) * e.cols;
    const S *g = static_cast<const S *>(e.g) + elems * which;
    const float *mom = e.mom ? e.mom + elems * which : nullptr;
    const bool flip = e.rows > e.cols;
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    // row r and columns c.. of this tile as it lies in U
    const int ur = (flip ? n0 : m0) + r, uc = (flip ? m0 : n0) + c;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        float u = 0.0f;
        if (ur < e.rows && uc + k < e.cols) {
            const size_t at = static_cast<size_t>(ur) * e.cols + uc + k;
            u = static_cast<float>(g[at]);
            if (mom) u = update_of(u, mom[at], p);
            u = static_cast<float>(u * scale);
        }
        v[k] = u;
    }
    if (flip) {
#pragma unroll
        for (int k = 0; k < 16; ++k) tile[c + k][r] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = tile[r][c + k];
    }
    half8 hi[2], lo[2];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const _Float16 h = static_cast<_Float16>(v[k]);
        hi[k / 8][k % 8] = h;
        lo[k / 8][k % 8] = static_cast<_Float16>(v[k] - static_cast<float>(h));
    }
    _Float16 *x = q.x0 + static_cast<size_t>(m0 + r) * e.np + n0 + c;
    half8 *xh = reinterpret_cast<half8 *>(x), *xl = reinterpret_cast<half8 *>(x + q.xs);
    xh[0] = hi[0];
    xh[1] = hi[1];
    xl[0] = lo[0];
    xl[1] = lo[1];
}

enum { kGram = 0, kPoly = 1, kApply = 2 };

struct MuonStage {
    int cur;       // which X is read
    int full;      // P needs its lo part
    int last;      // the step's result goes to the caller
    DType wt;
    float a, b, c, decay;
};

// One product stage. A workgroup computes BM x BN of it: the M side's rows (of X, A or P) lie along the sum in memory
// and so do the N side's of kGram and kPoly, which multiply by a transpose; kApply's N side is X itself, whose
// fragments are transposed on their way out of LDS. Both sides travel straight to LDS, 128 bytes a row: 64 of the sum,
// or 32 with both parts. Rows are swizzled so that a fragment's 16-byte reads spread over the banks.
// The MFMA's first operand is the N side: a lane then holds 4 neighbouring columns of one row.
template<int KIND, int BM, int BN, bool SPLIT>
__global__ __launch_bounds__(256, 2) void k_muon_product(MuonTable t, MuonStage st) {
    constexpr int WM = BM / 2, WN = BN / 2, MT = WM / 32, NT = WN / 32;
    constexpr int BK = SPLIT ? 32 : 64;
    constexpr bool NN = KIND == kApply;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][(BM + BN) * 128];

    const int per_xcd = gridDim.x / 8; // workgroups of one matrix next to each other on one chiplet's L2
    const int blk = static_cast<int>(blockIdx.x) < per_xcd * 8 ? (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3)
                                                                 : static_cast<int>(blockIdx.x);
    const int i = entry_of(t, blk);
    const MuonEntry &e = t.e[i];
    const int tm = (e.mp + BM - 1) / BM, tn = NN ? (e.np + BN - 1) / BN : tm;
    const int tiles = NN ? tm * tn : tm * (tm + 1) / 2;
    const int b = blk - t.first[i], which = b / tiles;
    int ti, tj;
    if constexpr (NN) {
        ti = b % tiles % tm;
        tj = b % tiles / tm;
    } else { // tiles on and above the diagonal
        int rest = b % tiles;
        ti = 0;
        while (rest >= tm - ti) rest -= tm - ti++;
        tj = ti + rest;
    }
    const Planes q = planes_of(t.ws, e, which);
    const _Float16 *x = st.cur ? q.x1 : q.x0;
    _Float16 *xn = st.cur ? q.x0 : q.x1;
    const int m0 = ti * BM, n0 = tj * BN;
    const int K = KIND == kGram ? e.np : e.mp;
    const _Float16 *ms = KIND == kGram ? x : KIND == kPoly ? q.a : q.p;
    const _Float16 *ns = KIND == kPoly ? q.a : x;
    const size_t mps = KIND == kGram ? q.xs : q.as, nps = KIND == kPoly ? q.as : q.xs;
    const int mld = K, nld = NN ? e.np : K;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // source of each 16-byte piece this lane brings to LDS; rows and columns past the matrix repeat its last ones
    constexpr int MI = BM / 32, NI = BN / 32;
    const _Float16 *mp[MI], *np[NI];
#pragma unroll
    for (int k = 0; k < MI; ++k) {
        const int r = (wave * MI + k) * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
        const int gr = m0 + r < e.mp ? m0 + r : e.mp - 1;
        mp[k] = ms + (SPLIT ? (c >> 2) * mps + (c & 3) * 8 : c * 8) + static_cast<size_t>(gr) * mld;
    }
    constexpr int LPR = BN / 8; // lanes per row of the N side of kApply
    constexpr int SWZ = BN == 128 ? 2 : 1;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        if constexpr (NN) {
            const int r = (wave * NI + k) * (64 / LPR) + lane / LPR, c = (lane % LPR) ^ ((r & 3) << SWZ);
            const int gc = n0 + c * 8 < e.np ? n0 + c * 8 : e.np - 8;
            np[k] = ns + (SPLIT ? (r >> 5) * nps + static_cast<size_t>(r & 31) * nld : static_cast<size_t>(r) * nld) + gc;
        } else {
            const int r = (wave * NI + k) * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
            const int gr = n0 + r < e.mp ? n0 + r : e.mp - 1;
            np[k] = ns + (SPLIT ? (c >> 2) * nps + (c & 3) * 8 : c * 8) + static_cast<size_t>(gr) * nld;
        }
    }
    const size_t nstep = NN ? static_cast<size_t>(BK) * nld : BK;
    const auto fetch = [&](int buf) {
        uint8_t *to = lds[buf];
#pragma unroll
        for (int k = 0; k < MI; ++k) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)mp[k],
                                             (__attribute__((address_space(3))) void *)(to + (wave * MI + k) * 1024), 16,
                                             0, 0);
            mp[k] += BK;
        }
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)np[k],
                (__attribute__((address_space(3))) void *)(to + BM * 128 + (wave * NI + k) * 1024), 16, 0, 0);
            np[k] += nstep;
        }
    };

    const int wm = (wave & 1) * WM, wn = (wave >> 1) * WN;
    const int half = lane >> 5, l32 = lane & 31;
    float16v acc[NT][MT] = {};
    fetch(0);
    for (int k0 = 0, buf = 0; k0 < K; k0 += BK, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads(); // the tile has landed, and the other buffer's readers are done
        const uint8_t *ml = lds[buf], *nl = lds[buf] + BM * 128;
        half8 mf[MT][4], nf[NT][4]; // four pieces of 16 of the sum: hi 0, 1 and lo 0, 1, or 0..3
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                const int r = wm + u * 32 + l32;
                mf[u][s] = *reinterpret_cast<const half8 *>(ml + r * 128 + (((2 * s + half) ^ (r & 7)) << 4));
            }
#pragma unroll
            for (int y = 0; y < NT; ++y) {
                if constexpr (NN) {
                    const int l16 = lane & 15;
                    const int col = wn + y * 32 + ((lane >> 4) & 1) * 16 + (l16 & 3) * 4;
                    half4 h[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const int r = 16 * s + 8 * half + 4 * z + (l16 >> 2);
                        const uint8_t *at = nl + r * (BN * 2) + (((col >> 3) ^ ((r & 3) << SWZ)) << 4) + (col & 7) * 2;
                        h[z] = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                             (__attribute__((address_space(3))) short4v *)at));
                    }
                    nf[y][s] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
                } else {
                    const int r = wn + y * 32 + l32;
                    nf[y][s] = *reinterpret_cast<const half8 *>(nl + r * 128 + (((2 * s + half) ^ (r & 7)) << 4));
                }
            }
        }
        if (k0 + BK < K) fetch(buf ^ 1);
        const auto mul = [&](int sn, int sm) {
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
                for (int u = 0; u < MT; ++u)
                    acc[y][u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(nf[y][sn], mf[u][sm], acc[y][u], 0, 0, 0);
        };
        if constexpr (SPLIT) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                mul(s, s);
                mul(s, s + 2);
                mul(s + 2, s);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) mul(s, s);
        }
    }

    const auto split = [](float v, _Float16 &h, _Float16 &l) {
        h = static_cast<_Float16>(v);
        l = static_cast<_Float16>(v - static_cast<float>(h));
    };
    const bool flip = e.rows > e.cols;
    const int small = flip ? e.cols : e.rows, large = flip ? e.rows : e.cols;
#pragma unroll
    for (int y = 0; y < NT; ++y) {
#pragma unroll
        for (int u = 0; u < MT; ++u) {
            const int mb = m0 + wm + u * 32, nb = n0 + wn + y * 32;
            if (mb >= e.mp || nb >= (NN ? e.np : e.mp)) continue;
            const int m = mb + l32;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int n = nb + 8 * k + 4 * half;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[y][u][4 * k + r];
                if constexpr (KIND == kApply) {
                    const size_t at = static_cast<size_t>(m) * e.np + n;
                    const half4 xh = *reinterpret_cast<const half4 *>(x + at);
                    const half4 xl = *reinterpret_cast<const half4 *>(x + q.xs + at);
                    half4 oh, ol;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        v[r] = v[r] * (1.0f / kMuonScaleP) +
                               st.a * (static_cast<float>(xh[r]) + static_cast<float>(xl[r]));
                        _Float16 h, l;
                        split(v[r], h, l);
                        oh[r] = h;
                        ol[r] = l;
                    }
                    if (!st.last) {
                        *reinterpret_cast<half4 *>(xn + at) = oh;
                        *reinterpret_cast<half4 *>(xn + q.xs + at) = ol;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (m >= small || n + r >= large) continue;
                            const size_t o = static_cast<size_t>(e.rows) * e.cols * which +
                                             (flip ? static_cast<size_t>(n + r) * e.cols + m
                                                   : static_cast<size_t>(m) * e.cols + n + r);
                            float out = v[r] * (1.0f / kMuonScaleX);
                            if (e.mom) out = load_as(e.w, o, st.wt) * st.decay - e.alpha * out;
                            store_as(e.w, o, st.wt, out);
                        }
                    }
                } else {
                    const size_t at = static_cast<size_t>(m) * e.mp + n;
                    _Float16 *to = KIND == kGram ? q.a : q.p;
                    half4 oh, ol;
                    if constexpr (KIND == kGram) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] *= kMuonScaleA / (kMuonScaleX * kMuonScaleX);
                    } else {
                        const half4 ah = *reinterpret_cast<const half4 *>(q.a + at);
                        const half4 al = *reinterpret_cast<const half4 *>(q.a + q.as + at);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            v[r] = v[r] * (st.c * (kMuonScaleP / (kMuonScaleA * kMuonScaleA))) +
                                   (st.b * (kMuonScaleP / kMuonScaleA)) *
                                       (static_cast<float>(ah[r]) + static_cast<float>(al[r]));
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        _Float16 h, l;
                        split(v[r], h, l);
                        oh[r] = h;
                        ol[r] = l;
                    }
                    const bool lows = KIND == kGram || st.full;
                    *reinterpret_cast<half4 *>(to + at) = oh;
                    if (lows) *reinterpret_cast<half4 *>(to + q.as + at) = ol;
                    if (ti != tj) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const size_t mt = static_cast<size_t>(n + r) * e.mp + m;
                            to[mt] = oh[r];
                            if (lows) to[q.as + mt] = ol[r];
                        }
                    }
                }
            }
        }
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

template<int KIND, int BM, int BN>
bool launch_product(MuonTable &t, const MuonStage &st, bool split, hipStream_t s) {
    const int64_t n = layout(t, [](const MuonEntry &e) {
        const int64_t tm = (e.mp + BM - 1) / BM;
        return KIND == kApply ? tm * ((e.np + BN - 1) / BN) : tm * (tm + 1) / 2;
    });
    if (n > INT32_MAX) return false;
    const dim3 grid(static_cast<unsigned>(n));
    return launch_ok([&] {
        if (split)
            k_muon_product<KIND, BM, BN, true><<<grid, 256, 0, s>>>(t, st);
        else if constexpr (KIND != kPoly)
            k_muon_product<KIND, BM, BN, false><<<grid, 256, 0, s>>>(t, st);
    });
}

template<int KIND>
bool launch_stage(MuonTable &t, const MuonStage &st, bool split, hipStream_t s) {
    int64_t big = 0;
    for (int i = 0; i < t.n; ++i) {
        const int64_t tm = (t.e[i].mp + 127) / 128;
        big += t.e[i].count * (KIND == kApply ? tm * ((t.e[i].np + 127) / 128) : tm * (tm + 1) / 2);
    }
    if (big >= 256) return launch_product<KIND, 128, 128>(t, st, split, s);
    return launch_product<KIND, 64, 64>(t, st, split, s);
}

} // namespace

bool launch_muon(const MuonEntry *entries, int n, DType gt, DType wt, const MuonParams &p, void *ws, hipStream_t s) {
    MuonTable t{};
    t.ws = static_cast<uint8_t *>(ws);
    t.n = n;
    for (int i = 0; i < n; ++i) t.e[i] = entries[i];
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
        int64_t blocks = layout(t, [](const MuonEntry &e) { return e.partials; });
        if (blocks > INT32_MAX) return false;
        if (!launch_ok([&] { k_muon_momentum<G><<<dim3(static_cast<unsigned>(blocks)), 256, 0, s>>>(t, p); }))
            return false;
        blocks = layout(t, [](const MuonEntry &e) { return static_cast<int64_t>(e.mp / 64) * (e.np / 64); });
        if (blocks > INT32_MAX) return false;
        return launch_ok([&] { k_muon_start<G><<<dim3(static_cast<unsigned>(blocks)), 256, 0, s>>>(t, p); });
    });
    if (!started) return false;
    const bool split = wt != DType::BF16;
    for (int k = 0; k < p.steps; ++k) {
        const MuonStage st{k & 1, split ? 1 : 0, k == p.steps - 1 ? 1 : 0, wt, p.a, p.b, p.c, p.decay};
        if (!launch_stage<kGram>(t, st, split, s) || !launch_stage<kPoly>(t, st, true, s) ||
            !launch_stage<kApply>(t, st, split, s))
            return false;
    }
    return true;
}

} // namespace pccl::hipk
