// Log probabilities of given tokens with entropy and top alternatives, and their gradient (formulas in
// csrc/kernels/logprob_common.hpp).
//
// Memory bound: the forward reads every logit once, the backward reads and writes each once. One workgroup per row
// holds a running (max, sum of exponentials, sum of exponentials times distance) per thread in fp32 and joins them at
// the end, so the row is never stored in a wider type. The sums' order is fixed by row length and workgroup size, so
// equal calls give equal bits. 12288 x 50304 bf16: forward 210 us, 5.9 TB/s (with 20 alternatives 239 us); backward
// 466 us, 5.3 TB/s; a large copy moves 4.8 TB/s. One row of 50304 takes 7 us, 10 with alternatives, where a call's
// host side takes 13 to 17: a row is not split over workgroups.
//
// Top alternatives need no second pass over the row: each thread also knows its best value and the block of the row
// where it first stood, and 64 groups of threads the best of these. Ordered by (value, earlier block), the k-th best of
// the 64 pairs bounds the k best elements from below -- each of the k better groups has an element that beats everything
// in a group behind it -- so only threads of k groups have their elements looked at again.
#include <algorithm>

#include "dispatch.hpp"
#include "launchers.hpp"

namespace pccl::hipk {

using kernels::kMaxTopLogprobs;
using kernels::LogprobArgs;
using kernels::LogprobGradArgs;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kUnroll = 4;      // 16-byte loads in flight per thread
constexpr int kCandidates = 1024;
constexpr int64_t kRowsPerLaunch = 1 << 22; // a launch has fewer than 2^32 threads

// storage types with the hardware conversions (round to nearest even)
struct LF32 {
    using S = float;
    static __device__ __forceinline__ float ld(S v) { return v; }
    static __device__ __forceinline__ S st(float v) { return v; }
};
struct LBF16 {
    using S = __bf16;
    static __device__ __forceinline__ float ld(S v) { return static_cast<float>(v); }
    static __device__ __forceinline__ S st(float v) { return static_cast<__bf16>(v); }
};
struct LF16 {
    using S = _Float16;
    static __device__ __forceinline__ float ld(S v) { return static_cast<float>(v); }
    static __device__ __forceinline__ S st(float v) { return static_cast<_Float16>(v); }
};

// 16 bytes at any element alignment (rows of an odd vocabulary, views that skip padded columns)
template<typename S>
struct __attribute__((packed, aligned(sizeof(S)))) Block {
    S v[16 / sizeof(S)];
};

template<typename E>
__device__ __forceinline__ void load_block(const typename E::S *x, int64_t b, int64_t full, int64_t vocab,
                                           float (&v)[16 / sizeof(typename E::S)]) {
    using S = typename E::S;
    constexpr int W = 16 / sizeof(S);
    if (b < full) {
        const Block<S> t = *reinterpret_cast<const Block<S> *>(x + b * W);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = E::ld(t.v[i]);
    } else { // the last, partial block, and none
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = b * W + i < vocab ? E::ld(x[b * W + i]) : kNegInf;
    }
}

// order of the alternatives: larger value first; equal zeros are equal, NaN stands with -inf
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x != x ? kNegInf : x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t pair_key(uint32_t key, uint32_t pos) {
    return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - pos);
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// k-th largest of a wave's 64 keys, 0 if fewer than k are non-zero: bit by bit over the values, then over the positions
// of those that share the k-th value
__device__ uint64_t kth_largest(uint64_t key, int k) {
    const uint32_t kh = static_cast<uint32_t>(key >> 32), kl = static_cast<uint32_t>(key);
    uint32_t hi = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = hi | (1u << bit);
        if (__popcll(__ballot(kh >= c)) >= k) hi = c;
    }
    if (hi == 0) return 0;
    const int need = k - __popcll(__ballot(kh > hi));
    if (__popcll(__ballot(kh == hi)) == need) return static_cast<uint64_t>(hi) << 32;
    uint32_t lo = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = lo | (1u << bit);
        if (__popcll(__ballot(kh == hi && kl >= c)) >= need) lo = c;
    }
    return (static_cast<uint64_t>(hi) << 32) | lo;
}

struct RowSums {
    float m, s, t; // max, sum exp(x - m), sum exp(x - m) (x - m)
};
// (x - m) for the exponential's factor: a masked entry's -inf must not meet its zero weight
__device__ __forceinline__ float bounded(float d) { return __builtin_fmaxf(d, -200.0f); }
__device__ __forceinline__ RowSums join(const RowSums &a, const RowSums &b) {
    const float m = __builtin_fmaxf(a.m, b.m);
    const float mu = m == kNegInf ? 0.0f : m;
    const float ea = __builtin_amdgcn_exp2f((a.m - mu) * kLog2e), eb = __builtin_amdgcn_exp2f((b.m - mu) * kLog2e);
    return {m, a.s * ea + b.s * eb, ea * (a.t + bounded(a.m - mu) * a.s) + eb * (b.t + bounded(b.m - mu) * b.s)};
}

} // namespace

template<typename E, int T, bool TOP>
__global__ __launch_bounds__(T) void k_token_logprob(LogprobArgs a) {
    using S = typename E::S;
    constexpr int W = 16 / sizeof(S);
    constexpr int kWaves = T / 64;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const S *x = static_cast<const S *>(a.logits) + row * a.row_stride;
    const int64_t full = a.vocab / W, blocks = (a.vocab + W - 1) / W;

    RowSums r{kNegInf, 0.0f, 0.0f};
    uint32_t best = tid; // block of the row where this thread's maximum first stood
    const auto add = [&](auto &v, uint32_t b0) { // blocks b0, b0 + T, .. of this thread
        constexpr int N = sizeof(v) / sizeof(v[0]);
        float nm = r.m;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            float bm = v[u][0];
#pragma unroll
            for (int i = 1; i < W; ++i) bm = __builtin_fmaxf(bm, v[u][i]);
            if constexpr (TOP) best = bm > nm ? b0 + u * T : best;
            nm = __builtin_fmaxf(nm, bm);
        }
        const float mu = nm == kNegInf ? 0.0f : nm;
        const float dm = r.m - mu;
        const float sc = __builtin_amdgcn_exp2f(dm * kLog2e);
        float s = r.s * sc, t = sc * (r.t + bounded(dm) * r.s);
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float d = v[u][i] - mu;
                const float e = __builtin_amdgcn_exp2f(d * kLog2e); // NaN logits reach the sum here
                s += e;
                t = __builtin_fmaf(e, bounded(d), t);
            }
        r = {nm, s, t};
    };
    int64_t b0 = 0;
    for (; b0 + kUnroll * T <= full; b0 += kUnroll * T) { // every thread has all its blocks: loads first, no branch
        Block<S> raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) raw[u] = *reinterpret_cast<const Block<S> *>(x + (b0 + u * T + tid) * W);
        float v[kUnroll][W];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) v[u][i] = E::ld(raw[u].v[i]);
        add(v, static_cast<uint32_t>(b0 + tid));
    }
    for (int64_t b = b0 + tid; b < blocks; b += T) {
        float v[1][W];
        load_block<E>(x, b, full, a.vocab, v[0]);
        add(v, static_cast<uint32_t>(b));
    }
    const RowSums mine = r;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        r = join(r, {__shfl_xor(r.m, o), __shfl_xor(r.s, o), __shfl_xor(r.t, o)});
    if constexpr (kWaves > 1) {
        __shared__ RowSums part[kWaves];
        if ((tid & 63) == 0) part[tid >> 6] = r;
        __syncthreads();
        r = part[0];
#pragma unroll 1
        for (int w = 1; w < kWaves; ++w) r = join(r, part[w]);
    }
    const bool empty = r.m == kNegInf && r.s == 0.0f;
    const float L = empty ? 0.0f : logf(r.s);
    const auto logprob_of = [&](float v) { return empty ? kNegInf : (v - r.m) - L; };
    if (tid == 0) {
        const float H = empty ? 0.0f : L - r.t / r.s;
        a.stats[3 * row] = r.m;
        a.stats[3 * row + 1] = L;
        a.stats[3 * row + 2] = H;
        a.entropy[row] = H;
        const int64_t t = a.targets[row];
        float lp = 0.0f;
        if (t != a.ignore_index)
            lp = t >= 0 && t < a.vocab ? logprob_of(E::ld(x[t])) : __builtin_nanf("");
        a.logprob[row] = lp;
    }
    if constexpr (TOP) {
        __shared__ uint64_t keys[64];
        __shared__ uint64_t cand[kCandidates];
        __shared__ uint64_t bound;
        __shared__ int count, looking;
        __shared__ uint16_t lookers[T];
        const int k = a.top_k;
        const uint64_t own = tid < blocks ? pair_key(order_key(mine.m), best) : 0;
        uint64_t key = own;
#pragma unroll
        for (int o = 1; o < kWaves; o <<= 1) { // of a group of T / 64 neighbouring threads
            const uint64_t q = __shfl_xor(static_cast<unsigned long long>(key), o);
            key = q > key ? q : key;
        }
        if (tid % kWaves == 0) keys[tid / kWaves] = key;
        __syncthreads();
        if (tid < 64) {
            const uint64_t b = kth_largest(keys[tid], k);
            if (tid == 0) {
                bound = b;
                count = 0;
                looking = 0;
            }
        }
        __syncthreads();
        const uint64_t bd = bound;
        const bool looks = own != 0 && own >= bd;
        if (looks) lookers[atomicAdd(&looking, 1)] = tid;
        __syncthreads();
        // the lookers' blocks, shared out over the workgroup; the orders of arrival are lost in the ranks below
        const int nl = looking, per = static_cast<int>((blocks + T - 1) / T);
        for (int j = tid; j < nl * per; j += T) {
            const int64_t b = lookers[j % nl] + static_cast<int64_t>(j / nl) * T;
            if (b >= blocks) continue;
            float v[W];
            load_block<E>(x, b, full, a.vocab, v);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const uint32_t ek = order_key(v[i]);
                if (b * W + i >= a.vocab || pair_key(ek, static_cast<uint32_t>(b)) < bd) continue;
                const int at = atomicAdd(&count, 1);
                if (at < kCandidates) cand[at] = pair_key(ek, static_cast<uint32_t>(b * W + i));
            }
        }
        __syncthreads();
        const int n = count;
        auto put = [&](int rank, uint64_t c) {
            const uint32_t idx = 0xffffffffu - static_cast<uint32_t>(c);
            a.top_index[row * k + rank] = idx;
            a.top_logprob[row * k + rank] = logprob_of(value_of(static_cast<uint32_t>(c >> 32)));
        };
        if (n <= kCandidates) { // about k..3k of them, unless a thread holds many of the row's largest
            for (int i = tid; i < n; i += T) {
                const uint64_t c = cand[i];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) rank += cand[j] > c;
                if (rank < k) put(rank, c);
            }
        } else { // one alternative a round, the largest behind the last one
            __shared__ uint64_t wave_best[kWaves];
            uint64_t last = ~0ull;
            for (int rank = 0; rank < k; ++rank) {
                uint64_t c = 0;
                if (looks)
                    for (int64_t b = tid; b < blocks; b += T) {
                        float v[W];
                        load_block<E>(x, b, full, a.vocab, v);
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            if (b * W + i >= a.vocab) break;
                            const uint64_t e = pair_key(order_key(v[i]), static_cast<uint32_t>(b * W + i));
                            if (e < last && e > c) c = e;
                        }
                    }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    const uint64_t q = __shfl_xor(static_cast<unsigned long long>(c), o);
                    c = q > c ? q : c;
                }
                if ((tid & 63) == 0) wave_best[tid >> 6] = c;
                __syncthreads();
                c = wave_best[0];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) c = wave_best[w] > c ? wave_best[w] : c;
                __syncthreads();
                if (tid == 0) put(rank, c);
                last = c;
            }
        }
    }
}

// One pass: read a logit, write its gradient. Every workgroup owns `cols` columns of one row; the few columns of the
// target and the alternatives are written a second time, with their upstream gradient, by one thread each.
template<typename E, int T>
__global__ __launch_bounds__(T) void k_token_logprob_grad(LogprobGradArgs g, int64_t cols) {
    using S = typename E::S;
    constexpr int W = 16 / sizeof(S);
    const LogprobArgs &a = g.fwd;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int64_t c0 = blockIdx.y * cols, c1 = c0 + cols < a.vocab ? c0 + cols : a.vocab;
    const S *x = static_cast<const S *>(a.logits) + row * a.row_stride;
    S *out = static_cast<S *>(g.d_logits) + row * a.vocab;

    const float M = a.stats[3 * row], L = a.stats[3 * row + 1], H = a.stats[3 * row + 2];
    const bool empty = M == kNegInf && L == 0.0f;
    const int64_t target = a.targets[row];
    const bool has_target = target != a.ignore_index && g.g_logprob != nullptr;
    const float g_lp = has_target ? g.g_logprob[row] : 0.0f;
    const float gh = g.g_entropy ? g.g_entropy[row] : 0.0f;
    float gs = g_lp;
    if (g.g_top)
        for (int k = 0; k < a.top_k; ++k) gs += g.g_top[row * a.top_k + k];
    if (has_target && (target < 0 || target >= a.vocab)) gs = __builtin_nanf(""); // an invalid target is loud here too
    const float ghH = gh * H;
    const auto grad = [&](float v) {
        const float lp = (v - M) - L;
        const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
        return empty ? 0.0f : -p * (gs + __builtin_fmaf(gh, bounded(lp), ghH));
    };

    const int64_t n = c1 - c0, full = n / W;
    for (int64_t b0 = tid; b0 < full; b0 += static_cast<int64_t>(T) * kUnroll) {
        Block<S> in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (b0 + u * T < full) in[u] = *reinterpret_cast<const Block<S> *>(x + c0 + (b0 + u * T) * W);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (b0 + u * T >= full) break;
            Block<S> o;
#pragma unroll
            for (int i = 0; i < W; ++i) o.v[i] = E::st(grad(E::ld(in[u].v[i])));
            *reinterpret_cast<Block<S> *>(out + c0 + (b0 + u * T) * W) = o;
        }
    }
    for (int64_t i = c0 + full * W + tid; i < c1; i += T) out[i] = E::st(grad(E::ld(x[i])));
    if (empty) return;
    __syncthreads(); // the columns below were written above by other threads
    const int nk = g.g_top ? a.top_k : 0;
    if (tid <= nk) {
        int64_t j = target;
        float add = g_lp;
        bool mine = has_target;
        if (tid < nk) { // an alternative; it carries the target's gradient where they are one
            j = a.top_index[row * a.top_k + tid];
            add = g.g_top[row * a.top_k + tid] + (has_target && j == target ? g_lp : 0.0f);
            mine = true;
        } else {
            for (int k = 0; k < nk; ++k) mine = mine && a.top_index[row * a.top_k + k] != target;
        }
        if (mine && j >= c0 && j < c1) out[j] = E::st(grad(E::ld(x[j])) + add);
    }
}

// the n rows from r0 on
static LogprobArgs rows_of(LogprobArgs a, int64_t r0, int64_t n, size_t esize) {
    a.logits = static_cast<const uint8_t *>(a.logits) + esize * a.row_stride * r0;
    a.rows = n;
    a.targets += r0;
    a.stats += 3 * r0;
    if (a.logprob) a.logprob += r0;
    if (a.entropy) a.entropy += r0;
    if (a.top_logprob) a.top_logprob += r0 * a.top_k;
    if (a.top_index) a.top_index += r0 * a.top_k;
    return a;
}

template<typename F>
static bool with_logit(DType t, F &&f) {
    switch (t) {
        case DType::F32: return f(LF32{});
        case DType::BF16: return f(LBF16{});
        case DType::F16: return f(LF16{});
        default: return false;
    }
}

bool launch_token_logprobs(const LogprobArgs &a, DType t, hipStream_t st) {
    if (a.rows == 0) return true;
    if (a.rows > kRowsPerLaunch) {
        for (int64_t r = 0; r < a.rows; r += kRowsPerLaunch)
            if (!launch_token_logprobs(rows_of(a, r, std::min(kRowsPerLaunch, a.rows - r), dtype_size(t)), t, st))
                return false;
        return true;
    }
    return with_logit(t, [&](auto e) {
        using E = decltype(e);
        constexpr int W = 16 / sizeof(typename E::S);
        const dim3 grid(static_cast<unsigned>(a.rows));
        auto run = [&](auto threads) {
            constexpr int T = decltype(threads)::value;
            return launch_ok([&] {
                if (a.top_k > 0)
                    k_token_logprob<E, T, true><<<grid, T, 0, st>>>(a);
                else
                    k_token_logprob<E, T, false><<<grid, T, 0, st>>>(a);
            });
        };
        // Threads per row, by its 16-byte blocks alone: enough that a thread has few to look at again for the
        // alternatives, few enough that joining them costs little. 12288 rows, k = 0 / 20, in us with 64 / 128 / 256 /
        // 512 threads: bf16 x 512 (64 blocks) 8 11 20 46 / 20 24 216 242; bf16 x 5000 (625) 25 25 35 60 / 48 39 55 102;
        // bf16 x 16000 (2000) 84 83 78 111 / 134 115 98 146; bf16 x 50304 (6288) 234 237 225 220 / 444 364 279 239.
        // One row: bf16 x 50304 18 11 7.1 6.9 / 44 20 12 10 (1024 threads: 8.5 / 12).
        const int64_t blocks = (a.vocab + W - 1) / W;
        if (blocks <= 256) return run(std::integral_constant<int, 64>{});
        if (blocks <= 1024) return run(std::integral_constant<int, 128>{});
        if (blocks <= 3000) return run(std::integral_constant<int, 256>{});
        return run(std::integral_constant<int, 512>{});
    });
}

bool launch_token_logprobs_grad(const LogprobGradArgs &g, DType t, hipStream_t st) {
    if (g.fwd.rows == 0) return true;
    if (g.fwd.rows > kRowsPerLaunch) {
        for (int64_t r = 0; r < g.fwd.rows; r += kRowsPerLaunch) {
            LogprobGradArgs part = g;
            part.fwd = rows_of(g.fwd, r, std::min(kRowsPerLaunch, g.fwd.rows - r), dtype_size(t));
            if (g.g_logprob) part.g_logprob += r;
            if (g.g_entropy) part.g_entropy += r;
            if (g.g_top) part.g_top += r * g.fwd.top_k;
            part.d_logits = static_cast<uint8_t *>(g.d_logits) + dtype_size(t) * g.fwd.vocab * r;
            if (!launch_token_logprobs_grad(part, t, st)) return false;
        }
        return true;
    }
    return with_logit(t, [&](auto e) {
        using E = decltype(e);
        constexpr int T = 256;
        const int64_t per = T * kUnroll * static_cast<int64_t>(16 / sizeof(typename E::S)); // one sweep of a workgroup
        int64_t split = 1; // few rows: several workgroups share one
        while (g.fwd.rows * split < 1024 && split * per < g.fwd.vocab) ++split;
        const int64_t cols = ((g.fwd.vocab + split - 1) / split + per - 1) / per * per;
        const dim3 grid(static_cast<unsigned>(g.fwd.rows), static_cast<unsigned>((g.fwd.vocab + cols - 1) / cols));
        return launch_ok([&] { k_token_logprob_grad<E, T><<<grid, T, 0, st>>>(g, cols); });
    });
}

} // namespace pccl::hipk
