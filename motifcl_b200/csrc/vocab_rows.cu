// What rows of logits say about tokens: log probabilities of given tokens with the entropy of the row and its most probable
// tokens, the gradient of both, and the loss of a student against the tokens that a teacher kept, with its gradient.
//
// With T the temperature, m the largest logit of a row and d_c = (x_c - m) / T:
//     s = sum exp(d_c)      log p_c = d_c - ln s      H = ln s - (sum exp(d_c) d_c) / s
// so that both parts of H have one sign and nothing cancels.  m and s are kept apart (row_stats): their sum m / T + ln s would lose
// the last digits of every log p_c where the logits are large.  Exponentials are 2^(d log2 e): one product, one ex2.approx, 2 ulp.
// Masked logits (-infinity, the lowest float) and rows with nothing left fall out of one clamp: 2^-150 is 0 in fp32, and
// 0 * -150 is 0 where 0 * -infinity is not a number.
#include "kernels.h"

#include <cfloat>
#include <cmath>

namespace mcl {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxList = kVocabListMax;
constexpr int kMaxCluster = 8;
constexpr int kCandidates = 2048;      // above a row's threshold, before the exact selection
constexpr int kFinalists = 1024;       // a second threshold's
constexpr float kLn2 = 0.69314718f;    // ln 2 to fp32
static_assert(kMaxCluster * kMaxList <= kCandidates, "the lists of a cluster's CTAs are candidates of its first one");

// max(v, -150) that keeps NaN
__device__ __forceinline__ float clamp_low(float v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(-150.0f));
    return r;
}
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_top(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ---- running statistics of a part of a row -----------------------------------------------------------------------------
// c = log2(e) / T.  m: largest so far (the lowest float where nothing was above it), s: sum of e = 2^((x - m) c), a: sum of e (x - m) c.
template <bool ENTROPY>
struct Stats {
    float m = -FLT_MAX, s = 0.0f, a = 0.0f;
    __device__ __forceinline__ void raise(float to, float c) {
        const float d = clamp_low((m - to) * c), f = exp2_fast(d);
        if (ENTROPY) a = f * (a + d * s);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void term(float x, float c) {
        const float d = clamp_low((x - m) * c), e = exp2_fast(d);
        s += e;
        if (ENTROPY) a = fmaf(e, d, a);
    }
    __device__ __forceinline__ void add(float x, float c) {
        if (x > m) raise(x, c);
        term(x, c);
    }
    __device__ __forceinline__ void add(float4 v, float c) {
        const float top = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        if (top > m) raise(top, c);
        term(v.x, c); term(v.y, c); term(v.z, c); term(v.w, c);
    }
};

// ---- a CTA's part of a row: `head` scalars up to a 16-byte boundary, n4 quads, the rest as scalars -----------------------
struct Part {
    const float* p;
    int n, head, n4;
    __device__ __forceinline__ Part(const float* at, int count) : p(at), n(count) {
        head = (int)((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) >> 2;
        head = min(head, n);
        n4 = (n - head) >> 2;
    }
    __device__ __forceinline__ const float4* quads() const { return reinterpret_cast<const float4*>(p + head); }
    // f(quad's index, its values) for the quads of this thread, four of them in flight
    template <class F>
    __device__ __forceinline__ void each_quad(F f) const {
        constexpr int U = 4;
        int i = threadIdx.x;
        for (; i + (U - 1) * kRowThreads < n4; i += U * kRowThreads) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = load_behind(quads() + i + u * kRowThreads);
#pragma unroll
            for (int u = 0; u < U; ++u) f(i + u * kRowThreads, v[u]);
        }
        for (; i < n4; i += kRowThreads) f(i, load_behind(quads() + i));
    }
    // f(place, value) for the scalars around them
    template <class F>
    __device__ __forceinline__ void each_loose(F f) const {
        if ((int)threadIdx.x < n - 4 * n4) { const int at = loose(threadIdx.x); f(at, load_behind(p + at)); }
    }
    // place of the i-th scalar outside the quads, i < n - 4 n4
    __device__ __forceinline__ int loose(int i) const { return i < head ? i : i + 4 * n4; }
};

// ---- selection of the largest ------------------------------------------------------------------------------------------
// A candidate is one whole number: the logit's bits in an order that is the floats' (equal zeros equal), then the place, lower ones larger.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long candidate(float v, int at) {
    return (unsigned long long)ordered(v) << 32 | (0xffffffffu - (uint32_t)at);
}
struct Selection {
    unsigned long long list[kCandidates];
    unsigned long long last[kFinalists];
    unsigned long long best[kMaxList];     // largest first
    uint32_t bound[kRowWarps];
    int count, finalists, scanned[kRowWarps];
};
// A bound that at least k of the threads' values reach: every warp's r-th largest, r = k / warps rounded up, and of those the smallest.
// All threads; one barrier inside, one more before the next call.
__device__ __forceinline__ uint32_t bound_of(uint32_t mine, int k, uint32_t* bound) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t top = 0;
    for (int r = (k + kRowWarps - 1) / kRowWarps; r > 0; --r) {
        top = __reduce_max_sync(0xffffffffu, mine);
        const unsigned at = __ballot_sync(0xffffffffu, mine == top);
        if (lane == __ffs(at) - 1) mine = 0;
    }
    if (lane == 0) bound[warp] = top;
    __syncthreads();
    return __reduce_min_sync(0xffffffffu, bound[lane & (kRowWarps - 1)]);
}
// The k largest of list[0 .. n) to best[], in order; k <= n <= kCandidates.  All threads; ends with a barrier.
__device__ __forceinline__ void select_best(Selection& z, int n, int k) {
    const unsigned long long* from = z.list;
    int m = n;
    if (n > 2 * k) {                          // ranks cost n^2: first those below a bound go
        uint32_t mine = 0;
        for (int i = threadIdx.x; i < n; i += kRowThreads) mine = max(mine, (uint32_t)(z.list[i] >> 32));
        if (threadIdx.x == 0) z.finalists = 0;
        const uint32_t least = bound_of(mine, k, z.bound);       // 0 where threads without a candidate are among them
        for (int i = threadIdx.x; i < n; i += kRowThreads) {
            const unsigned long long v = z.list[i];
            if ((uint32_t)(v >> 32) < least) continue;
            const int at = atomicAdd(&z.finalists, 1);
            if (at < kFinalists) z.last[at] = v;
        }
        __syncthreads();
        if (z.finalists <= kFinalists) { from = z.last; m = z.finalists; }
    }
    for (int i = threadIdx.x; i < m; i += kRowThreads) {
        const unsigned long long v = from[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < m; ++j) rank += from[j] > v;         // no two are equal: their places differ
        if (rank < k) z.best[rank] = v;
    }
    __syncthreads();
}

// g[i] = f(x[i]) over a part; g may be x itself
template <class F>
__device__ __forceinline__ void write_part(const Part& part, float* g, F f) {
    if (((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(part.p)) & 15) == 0) {
        float4* g4 = reinterpret_cast<float4*>(g + part.head);
        part.each_quad([&](int i, float4 v) { g4[i] = make_float4(f(v.x), f(v.y), f(v.z), f(v.w)); });
    } else {
        float* gq = g + part.head;
        part.each_quad([&](int i, float4 v) { gq[4 * i] = f(v.x); gq[4 * i + 1] = f(v.y); gq[4 * i + 2] = f(v.z); gq[4 * i + 3] = f(v.w); });
    }
    part.each_loose([&](int at, float v) { g[at] = f(v); });
}
__device__ __forceinline__ void clear_part(float* g, int n) {
    const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) >> 2), n4 = (n - head) >> 2;
    for (int i = threadIdx.x; i < n4; i += kRowThreads) reinterpret_cast<float4*>(g + head)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if ((int)threadIdx.x < n - 4 * n4) g[(int)threadIdx.x < head ? threadIdx.x : threadIdx.x + 4 * n4] = 0.0f;
}

// ---- what a row's CTAs share -------------------------------------------------------------------------------------------
struct RowShared {
    float wm[kRowWarps], ws[kRowWarps], wa[kRowWarps];
    float cm[kMaxCluster], cs[kMaxCluster], ca[kMaxCluster];       // written by the cluster's CTAs
    float t[kMaxList], log_t[kMaxList], x[kMaxList];                // the teacher's list: probabilities, their logarithms, the student's logits there
    int id[kMaxList];                                               // -1: no entry
    float t_sum;                                                    // of the exponentials; 0: an empty list
};
__device__ __forceinline__ uint32_t cluster_address(const void* shared, int rank) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(shared)), "r"(rank));
    return to;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

struct VocabRows {
    const float* logits;
    size_t rows, stride;
    int cols, cluster;                 // CTAs of a row
    float c, inv_t;                    // log2(e) / T, 1 / T
    const int* tokens;                 // null: no log probabilities
    float* logprobs;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    int n_top;
    float* row_stats;
    const int* teacher_ids;
    const float* teacher_logits;
    int n_teacher;
    float* losses;
    const float* grad_out;             // with grad_logits
    float* grad_logits;
};

// The teacher's list of a row by one warp: probabilities of its entries among themselves, and the student's logits there.
__device__ __forceinline__ void read_list(const VocabRows& p, size_t row, RowShared& sh) {
    const int lane = threadIdx.x & 31;
    const float* x = p.logits + row * p.stride;
    const size_t at = row * (size_t)p.n_teacher;
    float top = -FLT_MAX, sum = 0.0f;
    for (int i = lane; i < p.n_teacher; i += 32) {
        const int id = load_behind(p.teacher_ids + at + i);
        const bool in = id >= 0 && id < p.cols;
        const float v = in ? load_behind(p.teacher_logits + at + i) : -INFINITY;
        sh.id[i] = in ? id : -1;
        sh.t[i] = sh.log_t[i] = v;
        sh.x[i] = in ? load_behind(x + id) : 0.0f;
        top = fmaxf(top, v);
    }
    top = warp_top(top);
    for (int i = lane; i < p.n_teacher; i += 32) sum += exp2_fast(clamp_low((sh.t[i] - top) * p.c));
    sum = warp_add(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, log_sum = logf(sum);
    if (lane == 0) sh.t_sum = sum;
    for (int i = lane; i < p.n_teacher; i += 32) {
        const float d = clamp_low((sh.t[i] - top) * p.c);
        sh.t[i] = exp2_fast(d) * inv;
        sh.log_t[i] = (sh.log_t[i] - top) * p.inv_t - log_sum;
    }
    __syncwarp();
}
// g[id] of the listed tokens in [c0, c0 + cn), behind the rest of g: the first entry that names one writes it, with all that name it, in their order
template <class F>
__device__ __forceinline__ void write_listed(const RowShared& sh, int n, float* g, int c0, int cn, float up, F value) {
    const int id = (int)threadIdx.x < n ? sh.id[threadIdx.x] : -1;
    if (id < c0 || id >= c0 + cn) return;
    float t = 0.0f;
    bool first = true;
    for (int j = 0; j < n; ++j)
        if (sh.id[j] == id) { t += sh.t[j]; first = first && j >= (int)threadIdx.x; }
    if (first) g[id - c0] = value(sh.x[threadIdx.x]) - t * up;
}

// One row at a time on a CTA, or a row on a cluster's CTAs where there are few.
template <bool ENTROPY, bool TOP, bool DISTILL>
__global__ void __launch_bounds__(kRowThreads) vocab_rows_kernel(VocabRows p) {
    grid_release();
    extern __shared__ __align__(16) unsigned char dynamic[];
    Selection& z = *reinterpret_cast<Selection*>(dynamic);       // TOP
    __shared__ RowShared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ranks = p.cluster, rank = ranks > 1 ? (int)(blockIdx.x % ranks) : 0;
    const int per = ((p.cols + ranks - 1) / ranks + 3) & ~3;
    const int c0 = min(p.cols, rank * per), cn = min(p.cols, c0 + per) - c0;
    if (ranks > 1) { cluster_arrive(); cluster_wait(); }          // every CTA of the cluster runs
    grid_wait();
    for (size_t row = blockIdx.x / ranks; row < p.rows; row += gridDim.x / ranks) {
        const float* x = p.logits + row * p.stride;
        const Part part(x + c0, cn);
        if (DISTILL && warp == 0) read_list(p, row, sh);
        float x_token = 0.0f;
        int token = -1;
        if (!DISTILL && p.tokens != nullptr && threadIdx.x == 0 && rank == 0) {
            token = load_behind(p.tokens + row);
            if (token < 0 || token >= p.cols) token = -1;
            else x_token = load_behind(x + token);
        }
        // the row's statistics
        Stats<ENTROPY> st;
        part.each_quad([&](int, float4 v) { st.add(v, p.c); });
        part.each_loose([&](int, float v) { st.add(v, p.c); });
        const float mine = st.m == -FLT_MAX ? -INFINITY : st.m;   // TOP: this thread's largest is no less
        float m = warp_top(st.m);
        if (lane == 0) sh.wm[warp] = m;
        __syncthreads();
        m = warp_top(sh.wm[lane & (kRowWarps - 1)]);
        st.raise(m, p.c);
        float s = warp_add(st.s), a = ENTROPY ? warp_add(st.a) : 0.0f;
        if (lane == 0) { sh.ws[warp] = s; if (ENTROPY) sh.wa[warp] = a; }
        __syncthreads();
        s = a = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) { s += sh.ws[w]; if (ENTROPY) a += sh.wa[w]; }
        if (ranks > 1) {
            if ((int)threadIdx.x < ranks) {
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(&sh.cm[rank], threadIdx.x)), "f"(m) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(&sh.cs[rank], threadIdx.x)), "f"(s) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(&sh.ca[rank], threadIdx.x)), "f"(a) : "memory");
            }
            cluster_arrive();
            cluster_wait();
            Stats<ENTROPY> all;
            for (int r = 0; r < ranks; ++r) all.m = fmaxf(all.m, sh.cm[r]);
            for (int r = 0; r < ranks; ++r) {
                Stats<ENTROPY> one;
                one.m = sh.cm[r]; one.s = sh.cs[r]; one.a = sh.ca[r];
                one.raise(all.m, p.c);
                all.s += one.s; all.a += one.a;
            }
            m = all.m; s = all.s; a = all.a;
        }
        const float log_s = logf(s);
        auto log_prob = [&](float v) { return s == 0.0f ? -INFINITY : (v - m) * p.inv_t - log_s; };      // s == 0: nothing is left of the row
        if (threadIdx.x == 0 && rank == 0) {
            if (p.row_stats != nullptr) { p.row_stats[2 * row] = m; p.row_stats[2 * row + 1] = s; }
            if (!DISTILL && p.logprobs != nullptr) p.logprobs[row] = token < 0 ? 0.0f : log_prob(x_token);
            if (ENTROPY && p.entropy != nullptr) p.entropy[row] = s == 0.0f ? 0.0f : log_s - a / s * kLn2;
        }
        if (TOP) {
            // Every thread has its largest; at least n_top of the row reach their bound.  What is above it is collected, equal ones are looked for
            // in order only where those are too few.  More than fit (values above the bound in few threads) give a higher bound.
            const int k = p.n_top, k_part = min(k, part.n);
            const bool nan = !(s == s);
            float over = unordered(max(bound_of(ordered(mine), k, z.bound), ordered(-INFINITY)));
            int n;
            for (;;) {
                __syncthreads();
                if (threadIdx.x == 0) z.count = 0;
                __syncthreads();
                auto look = [&](float v, int at) {
                    if (v > over) {
                        const int i = atomicAdd(&z.count, 1);
                        if (i < kCandidates) z.list[i] = candidate(v, c0 + at);
                    }
                };
                if (!nan) {
                    part.each_quad([&](int i, float4 v) {
                        if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) > over) {
                            const int at = part.head + 4 * i;
                            look(v.x, at); look(v.y, at + 1); look(v.z, at + 2); look(v.w, at + 3);
                        }
                    });
                    part.each_loose([&](int at, float v) { look(v, at); });
                }
                __syncthreads();
                n = z.count;
                if (n <= kCandidates) break;
                select_best(z, kCandidates, k);
                over = unordered((uint32_t)(z.best[k - 1] >> 32));
            }
            if (!nan && n < k_part) {                               // the lowest places of those equal to the bound
                for (int c = 0; c < part.n && n < k_part; c += kRowThreads) {
                    const int at = c + threadIdx.x;
                    const float v = at < part.n ? load_behind(part.p + at) : 0.0f;
                    const bool hit = at < part.n && v == over;
                    const unsigned hits = __ballot_sync(0xffffffffu, hit);
                    if (lane == 0) z.scanned[warp] = __popc(hits);
                    __syncthreads();
                    int before = n, all = n;
                    for (int w = 0; w < kRowWarps; ++w) { if (w < warp) before += z.scanned[w]; all += z.scanned[w]; }
                    before += __popc(hits & ((1u << lane) - 1));
                    if (hit && before < k_part) z.list[before] = candidate(v, c0 + at);
                    n = min(all, k_part);
                    __syncthreads();
                }
            }
            if (!nan) select_best(z, n, k_part);
            if (ranks > 1) {
                // the parts' lists are the candidates of the first CTA, which is behind its own selection when all have arrived
                cluster_arrive();
                cluster_wait();
                if ((int)threadIdx.x < k && !nan) {
                    const unsigned long long v = (int)threadIdx.x < k_part ? z.best[threadIdx.x] : 0ull;
                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_address(&z.list[rank * k + threadIdx.x], 0)), "l"(v) : "memory");
                }
                cluster_arrive();
                cluster_wait();
                // empty places (0) of parts shorter than k are below every candidate; they fall out by rank since cols >= k
                if (rank == 0 && !nan) {
                    if ((int)threadIdx.x < ranks * k && z.list[threadIdx.x] == 0ull) z.list[threadIdx.x] = threadIdx.x;
                    for (int i = threadIdx.x + kRowThreads; i < ranks * k; i += kRowThreads)
                        if (z.list[i] == 0ull) z.list[i] = i;        // unlike one another
                    __syncthreads();
                    select_best(z, ranks * k, k);
                }
            }
            if (rank == 0 && (int)threadIdx.x < k) {
                const unsigned long long v = nan ? 0ull : z.best[threadIdx.x];
                if (p.top_ids != nullptr) p.top_ids[row * k + threadIdx.x] = nan ? -1 : (int)(0xffffffffu - (uint32_t)v);
                if (p.top_logprobs != nullptr) p.top_logprobs[row * k + threadIdx.x] = nan ? s : log_prob(unordered((uint32_t)(v >> 32)));
            }
            __syncthreads();
        }
        if (DISTILL) {
            const float t_sum = sh.t_sum;
            if (warp == 0 && rank == 0 && p.losses != nullptr) {
                float loss = 0.0f;
                for (int i = lane; i < p.n_teacher; i += 32) {
                    const float t = sh.t[i];
                    if (t != 0.0f) loss += t * (sh.log_t[i] - log_prob(sh.x[i]));
                }
                loss = warp_add(loss);
                if (lane == 0) p.losses[row] = loss;
            }
            if (p.grad_logits != nullptr) {
                float* g = p.grad_logits + row * p.stride + c0;
                const float up = load_behind(p.grad_out) * p.inv_t / (float)p.rows;
                // an empty list or an empty row has no gradient; a list that is not a number has none that is one
                const bool none = t_sum == 0.0f || s == 0.0f;
                const float f = t_sum == t_sum ? up / s : t_sum;
                auto value = [&](float v) { return exp2_fast(clamp_low((v - m) * p.c)) * f; };
                if (none) clear_part(g, cn);
                else write_part(part, g, value);
                __syncthreads();
                if (!none) write_listed(sh, p.n_teacher, g, c0, cn, up, value);
            }
        }
        if (ranks > 1 && row + gridDim.x / ranks < p.rows) { cluster_arrive(); cluster_wait(); }
        __syncthreads();                                            // what the CTA shares is another row's from here on
    }
}

// ---- gradients from kept statistics ------------------------------------------------------------------------------------
struct VocabGrad {
    const float* logits;
    size_t rows, stride;
    int cols, tiles, per;              // tiles of a row, their length
    float c, inv_t;
    const float* row_stats;
    const int* tokens;
    const float* grad_logprobs;        // null: none
    const float* entropy;
    const float* grad_entropy;         // null: none
    const int* teacher_ids;
    const float* teacher_logits;
    int n_teacher;
    const float* grad_out;
    float* grad_logits;
};

// dx_c = e_c (k0 + k1 d_c) + (what the named tokens add), with e_c = 2^((x_c - m) c): p_c enters through 1 / s in k0 and k1.
template <bool DISTILL>
__global__ void __launch_bounds__(kRowThreads) vocab_grad_kernel(VocabGrad p) {
    grid_release();
    grid_wait();
    __shared__ RowShared sh;
    const size_t items = p.rows * (size_t)p.tiles;
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const size_t row = item / p.tiles;
        const int c0 = (int)(item - row * p.tiles) * p.per, cn = min(p.cols, c0 + p.per) - c0;
        const float* x = p.logits + row * p.stride;
        const Part part(x + c0, cn);
        float* g = p.grad_logits + row * p.stride + c0;
        const float m = load_behind(p.row_stats + 2 * row), s = load_behind(p.row_stats + 2 * row + 1);
        float k0 = 0.0f, k1 = 0.0f, up = 0.0f, x_token = 0.0f;
        int token = -1;
        bool none;
        if (DISTILL) {
            VocabRows list = {};
            list.logits = p.logits; list.stride = p.stride; list.cols = p.cols; list.c = p.c;
            list.teacher_ids = p.teacher_ids; list.teacher_logits = p.teacher_logits; list.n_teacher = p.n_teacher;
            if (threadIdx.x < 32) read_list(list, row, sh);
            __syncthreads();
            up = load_behind(p.grad_out) * p.inv_t / (float)p.rows;
            none = sh.t_sum == 0.0f;
            k0 = sh.t_sum == sh.t_sum ? up / s : sh.t_sum;
        } else {
            float h = 0.0f, H = 0.0f;
            if (p.grad_logprobs != nullptr) {
                token = load_behind(p.tokens + row);
                if (token < 0 || token >= p.cols) token = -1;
                else { up = load_behind(p.grad_logprobs + row) * p.inv_t; x_token = load_behind(x + token); }
            }
            if (p.grad_entropy != nullptr) { h = load_behind(p.grad_entropy + row) * p.inv_t; H = load_behind(p.entropy + row); }
            none = up == 0.0f && h == 0.0f;
            k0 = -(up + (h == 0.0f ? 0.0f : h * (H - logf(s)))) / s;
            k1 = -h * kLn2 / s;
            __syncthreads();                                        // x_token is read before it may be overwritten (grad_logits == logits)
        }
        none = none || s == 0.0f;
        auto value = [&](float v) {
            const float d = clamp_low((v - m) * p.c);
            return exp2_fast(d) * (DISTILL ? k0 : fmaf(k1, d, k0));
        };
        if (none) clear_part(g, cn);
        else write_part(part, g, value);
        __syncthreads();
        if (!none && DISTILL) write_listed(sh, p.n_teacher, g, c0, cn, up, value);
        if (!none && !DISTILL && threadIdx.x == 0 && token >= c0 && token < c0 + cn) g[token - c0] = value(x_token) + up;
        if (DISTILL) __syncthreads();                               // the list is another item's from here on
    }
}

// Attributes of a launch: overlapping with the one before it, and the CTAs of a row as a cluster.
template <class P>
cudaError_t launch_rows(void (*kern)(P), unsigned grid, int cluster, size_t smem, cudaStream_t stream, const P& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kRowThreads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}
// CTAs of a row: as many as leave none of the SMs idle, with 2048 logits each at least
int row_cluster(size_t rows, int cols, int sm_count) {
    int n = 1;
    while (n < kMaxCluster && rows * 2 * n <= 2 * (size_t)sm_count && cols / (2 * n) >= 2048) n *= 2;
    return n;
}
unsigned row_ctas(size_t rows, int cluster, int sm_count) {
    const size_t cap = (size_t)sm_count * 16 / cluster;
    return (unsigned)((rows < cap ? rows : cap) * cluster);
}
void temperature_of(float t, float* c, float* inv_t) {
    *inv_t = 1.0f / t;
    *c = (float)(1.4426950408889634 / (double)t);
}
cudaError_t launch_grad(bool distill, VocabGrad& p, int sm_count, cudaStream_t stream) {
    // tiles of a row where the rows are fewer than the CTAs that fill the SMs
    const size_t want = 4 * (size_t)sm_count;
    p.tiles = 1;
    while (p.rows * (size_t)p.tiles < want && p.cols / (2 * p.tiles) >= 2048) p.tiles *= 2;
    p.per = ((p.cols + p.tiles - 1) / p.tiles + 3) & ~3;
    p.tiles = (p.cols + p.per - 1) / p.per;
    const size_t items = p.rows * (size_t)p.tiles, cap = (size_t)sm_count * 16;
    return launch_rows(distill ? vocab_grad_kernel<true> : vocab_grad_kernel<false>, (unsigned)(items < cap ? items : cap), 1, 0, stream, p);
}
}  // namespace

cudaError_t launch_token_logprobs(const float* logits, const int* tokens, float* logprobs, float* entropy, int* top_ids, float* top_logprobs,
                                  float* row_stats, size_t rows, int cols, size_t stride, int n_top, float temperature, int sm_count,
                                  cudaStream_t stream) {
    VocabRows p = {};
    p.logits = logits; p.rows = rows; p.stride = stride; p.cols = cols;
    temperature_of(temperature, &p.c, &p.inv_t);
    p.tokens = tokens; p.logprobs = logprobs; p.entropy = entropy; p.top_ids = top_ids; p.top_logprobs = top_logprobs; p.n_top = n_top;
    p.row_stats = row_stats;
    p.cluster = row_cluster(rows, cols, sm_count);
    const unsigned grid = row_ctas(rows, p.cluster, sm_count);
    const size_t smem = n_top ? sizeof(Selection) : 0;
    if (n_top) return launch_rows(entropy ? vocab_rows_kernel<true, true, false> : vocab_rows_kernel<false, true, false>, grid, p.cluster, smem, stream, p);
    return launch_rows(entropy ? vocab_rows_kernel<true, false, false> : vocab_rows_kernel<false, false, false>, grid, p.cluster, smem, stream, p);
}
cudaError_t launch_token_logprobs_backward(const float* logits, const int* tokens, const float* row_stats, const float* entropy,
                                           const float* grad_logprobs, const float* grad_entropy, float* grad_logits, size_t rows, int cols,
                                           size_t stride, float temperature, int sm_count, cudaStream_t stream) {
    VocabGrad p = {};
    p.logits = logits; p.rows = rows; p.stride = stride; p.cols = cols;
    temperature_of(temperature, &p.c, &p.inv_t);
    p.row_stats = row_stats; p.tokens = tokens; p.grad_logprobs = grad_logprobs; p.entropy = entropy; p.grad_entropy = grad_entropy;
    p.grad_logits = grad_logits;
    return launch_grad(false, p, sm_count, stream);
}
cudaError_t launch_distillation_loss(const float* logits, const int* teacher_ids, const float* teacher_logits, float* losses, float* out,
                                     float* row_stats, const float* grad_out, float* grad_logits, size_t rows, int cols, size_t stride,
                                     int n_teacher, float temperature, int sm_count, cudaStream_t stream) {
    VocabRows p = {};
    p.logits = logits; p.rows = rows; p.stride = stride; p.cols = cols;
    temperature_of(temperature, &p.c, &p.inv_t);
    p.teacher_ids = teacher_ids; p.teacher_logits = teacher_logits; p.n_teacher = n_teacher;
    p.losses = losses; p.row_stats = row_stats; p.grad_out = grad_out; p.grad_logits = grad_logits;
    p.cluster = row_cluster(rows, cols, sm_count);
    const cudaError_t e = launch_rows(vocab_rows_kernel<false, false, true>, row_ctas(rows, p.cluster, sm_count), p.cluster, 0, stream, p);
    return e != cudaSuccess ? e : launch_mean(losses, out, rows, rows, stream);
}
cudaError_t launch_distillation_loss_backward(const float* logits, const int* teacher_ids, const float* teacher_logits, const float* row_stats,
                                              const float* grad_out, float* grad_logits, size_t rows, int cols, size_t stride, int n_teacher,
                                              float temperature, int sm_count, cudaStream_t stream) {
    VocabGrad p = {};
    p.logits = logits; p.rows = rows; p.stride = stride; p.cols = cols;
    temperature_of(temperature, &p.c, &p.inv_t);
    p.teacher_ids = teacher_ids; p.teacher_logits = teacher_logits; p.n_teacher = n_teacher; p.row_stats = row_stats;
    p.grad_out = grad_out; p.grad_logits = grad_logits;
    return launch_grad(true, p, sm_count, stream);
}
}  // namespace mcl
