// What rows of logits say about tokens: log probabilities of given tokens with the entropy of the row and its most probable
// tokens, the gradient of both, and the loss of a student against the tokens that a teacher kept, with its gradient.
//
// Bound by memory: a forward call reads the logits once, a gradient reads them and writes as much; next to that the issue slots, of which an fp32 value takes
// 11.8 thread-instructions where only its statistics are wanted (pairs of values an instruction) and 20.5 with the 20 largest sought.
// 4096 x 32000 (524 MB; at the rate of a copy its bytes take 81.5 us, 163 us read and written; a pass that only reads may be faster than that): log probabilities and entropy 78 us, with the 20 most probable
// tokens 110 us, their gradient 161 us; distillation from lists of 64: loss 80 us, loss and gradient in one call 184 us, gradient from kept statistics 176 us.
//
// With T the temperature, m the largest logit of a row and d_c = (x_c - m) / T:
//     s = sum exp(d_c)      log p_c = d_c - ln s      H = ln s - (sum exp(d_c) d_c) / s
// so that both parts of H have one sign and nothing cancels.  m and s are kept apart (row_stats): their sum m / T + ln s would lose
// the last digits of every log p_c where the logits are large.  Exponentials are 2^(d log2 e): one product, one ex2.approx, 2 ulp; below 2^-126 they are 0.
// log p_c takes (x_c - m) times the rounded 1 / T within the fma that takes ln s off: one rounding beside that of 1 / T, as many as a division would bring.
// Masked logits (-infinity, the lowest float) and rows with nothing left fall out of one clamp: 2^-150 is 0 in fp32, and
// 0 * -150 is 0 where 0 * -infinity is not a number.
#include "kernels.h"
#include "tc_ptx.cuh"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

namespace mcl {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kResultThread = kRowThreads - 32;        // writes a row's results: the first of the warp that has least to do at the end
constexpr int kQuads = 4;              // of a thread in a step
constexpr int kMaxList = kVocabListMax;
constexpr int kMaxCluster = 8;
constexpr int kHits = 928;             // quads with a value above a row's first bounds
constexpr int kCandidates = 512;       // values that reach its last one
constexpr float kLn2 = 0.69314718f;    // ln 2 to fp32

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

// Two fp32 values in one register pair: an instruction for both.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair_of(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float low_of(Pair v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high_of(Pair v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair clamp2(Pair v) { return pair_of(clamp_low(low_of(v)), clamp_low(high_of(v))); }
__device__ __forceinline__ Pair exp2_2(Pair v) { return pair_of(exp2_fast(low_of(v)), exp2_fast(high_of(v))); }

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
    // of the lanes xor 1 .. `lanes` / 2
    template <int LANES>
    __device__ __forceinline__ void join(float c) {
        float top = m;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        raise(top, c);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            if (ENTROPY) a += __shfl_xor_sync(0xffffffffu, a, o);
        }
    }
};
// The same while values go by, in two sums each.  Where there is no a to form, nothing needs a clamp: 2^-infinity is 0.
template <bool ENTROPY>
struct Running {
    float m = -FLT_MAX;
    Pair minus_m = pair_of(FLT_MAX, FLT_MAX), s = 0, a = 0;
    __device__ __forceinline__ void raise(float to, float c) {
        const float d = clamp_low((m - to) * c), f = exp2_fast(d);
        if (ENTROPY) a = mul2(fma2(pair_of(d, d), s, a), pair_of(f, f));
        s = mul2(s, pair_of(f, f));
        m = to;
        minus_m = pair_of(-to, -to);
    }
    __device__ __forceinline__ void terms(Pair x, float c) {
        Pair d = mul2(add2(x, minus_m), pair_of(c, c));
        if (ENTROPY) d = clamp2(d);
        const Pair e = exp2_2(d);
        s = add2(s, e);
        if (ENTROPY) a = fma2(e, d, a);
    }
    template <int N>
    __device__ __forceinline__ void quads(const float4 (&v)[N], float top, float c) {      // top: the largest of them
        if (top > m) raise(top, c);
#pragma unroll
        for (int u = 0; u < N; ++u) { terms(pair_of(v[u].x, v[u].y), c); terms(pair_of(v[u].z, v[u].w), c); }
    }
    __device__ __forceinline__ void one(float x, float c) {
        if (x > m) raise(x, c);
        terms(pair_of(x, -INFINITY), c);
    }
    __device__ __forceinline__ Stats<ENTROPY> sums() const {
        Stats<ENTROPY> r;
        r.m = m;
        r.s = low_of(s) + high_of(s);
        if (ENTROPY) r.a = low_of(a) + high_of(a);
        return r;
    }
    __device__ __forceinline__ float largest() const { return m == -FLT_MAX ? -INFINITY : m; }       // of what has gone by: no more than that
};
__device__ __forceinline__ float top_of(float4 v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }

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
    // place of the i-th scalar outside the quads, i < n - 4 n4
    __device__ __forceinline__ int loose(int i) const { return i < head ? i : i + 4 * n4; }
};

// The quads of a thread: those at threadIdx.x modulo the threads, kQuads of them a step, a quarter of the part apart, so that the first step is a
// sample of the part.  The distance depends on the part's length alone: a thread meets the same places whatever a row's alignment is.
__device__ __forceinline__ int quarter_of(int n, int threads) { return (((n >> 2) + kQuads - 1) / kQuads + threads - 1) / threads * threads; }
__device__ __forceinline__ void copy_async4(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Parts on their way: a thread copies the quads that it will work on itself, kAhead steps ahead and over the end of a part, so
// that nothing waits for another thread and memory is busy while a row is finished.  part(i): the i-th of `items`, of at most `longest` logits.
// With 4 CTAs an SM has 128 KB on their way.  4096 x 32000 alone / with 20 tops: 78 / 110 us; three steps ahead 84 / 138 (three CTAs an SM); half the threads,
// eight quads each 84 / 104 but 29 us instead of 27 for 777 x 50003; bulk copies and their barriers 81 / 117 (before the addresses were kept: 78 / 112).
constexpr int kAhead = 2;
template <int THREADS, class P>
struct Stream {
    // The addresses are kept, not formed anew for every copy: 112 us then for 4096 x 32000 with 20 tops, 108.5 so.
    static constexpr uint32_t kPlace = THREADS * 16, kSlot = kQuads * kPlace;
    const P& part;
    size_t next_item, items;
    const char* from;                  // this thread's first quad of the next step to fetch
    size_t stretch;                    // bytes of a quarter
    uint32_t mine, in, out;            // shared memory: this thread's place in the first slot; offsets of the slots to fill and to take
    int q, t, whole, n4;               // being fetched: its step, from which on a step is not whole, its quads
    __device__ __forceinline__ Stream(void* shared, const P& parts, size_t count, int longest)
        : part(parts), next_item(0), items(count), mine((uint32_t)__cvta_generic_to_shared(shared) + threadIdx.x * 16), in(0), out(0), q(quarter_of(longest, THREADS)) {
        stretch = (size_t)q * 16;
        if (q == 0) items = 0;
        start();
        for (int i = 0; i < kAhead; ++i) fetch();
    }
    __device__ __forceinline__ void start() {
        if (next_item >= items) return;
        const Part at = part(next_item);
        from = reinterpret_cast<const char*>(at.quads() + threadIdx.x);
        n4 = at.n4;
        t = 0;
        whole = at.n4 - (kQuads - 1) * q - THREADS;
    }
    template <int U>
    __device__ __forceinline__ void copy(uint32_t to, const char* at) {
        asm volatile("cp.async.cg.shared.global [%0+%2], [%1], 16;" ::"r"(to), "l"(at), "n"(U * (int)kPlace) : "memory");
    }
    template <int U>
    __device__ __forceinline__ void load(float4& v) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4+%5];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mine + out), "n"(U * (int)kPlace) : "memory");
    }
    __device__ __forceinline__ void fetch() {
        if (next_item < items) {
            const uint32_t to = mine + in;
            const char *b = from + stretch, *c = b + stretch, *d = c + stretch;
            if (t <= whole) {
                copy<0>(to, from); copy<1>(to, b); copy<2>(to, c); copy<3>(to, d);
            } else {
                const int i = t + (int)threadIdx.x;
                if (i < n4) copy<0>(to, from);
                if (i + q < n4) copy<1>(to, b);
                if (i + 2 * q < n4) copy<2>(to, c);
                if (i + 3 * q < n4) copy<3>(to, d);
            }
            from += THREADS * 16;
            t += THREADS;
            if (t >= q) { ++next_item; start(); }
        }
        copies_end();
        in = in + kSlot < kAhead * kSlot ? in + kSlot : 0;
    }
    // step `now` of a part with n4 quads: -infinity behind the end.  next() follows when the values have been used
    __device__ __forceinline__ void take(int now, int quads, float4 (&v)[kQuads]) {
        copies_wait<kAhead - 1>();
        load<0>(v[0]); load<1>(v[1]); load<2>(v[2]); load<3>(v[3]);
        out = out + kSlot < kAhead * kSlot ? out + kSlot : 0;
        if (now + (kQuads - 1) * q + THREADS <= quads) return;
#pragma unroll
        for (int u = 0; u < kQuads; ++u)
            if (u * q + now + (int)threadIdx.x >= quads) v[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
    __device__ __forceinline__ void next() { fetch(); }
};
static_assert(kQuads == 4, "a step's copies are written out");
constexpr size_t kStreamBytes = (size_t)kAhead * kQuads * kRowThreads * sizeof(float4);

// g[i] = f(x[i]) over a part; v is the first step, loaded by the caller ahead of what f waits for.  By loads and stores of the threads themselves:
// asynchronous copies behind stores wait in the same queue (4096 x 32000: 184 us, 161 so).
__device__ __forceinline__ void load_step(const Part& part, int q, int t, float4 (&v)[kQuads]) {
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
        const int i = u * q + t + (int)threadIdx.x;
        if (i < part.n4) v[u] = load_behind(part.quads() + i);
    }
}
// The gradients that f may be: f times p (1 / s is in f), and with the entropy's part e (k0 + k1 d).
struct ProbGrad {
    float m, c, f;
    __device__ __forceinline__ Pair operator()(Pair x) const { return mul2(exp2_2(mul2(add2(x, pair_of(-m, -m)), pair_of(c, c))), pair_of(f, f)); }
    __device__ __forceinline__ float operator()(float x) const { return exp2_fast((x - m) * c) * f; }
};
struct EntropyGrad {
    float m, c, k0, k1;
    __device__ __forceinline__ Pair operator()(Pair x) const {
        const Pair d = clamp2(mul2(add2(x, pair_of(-m, -m)), pair_of(c, c)));
        return mul2(exp2_2(d), fma2(pair_of(k1, k1), d, pair_of(k0, k0)));
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float d = clamp_low((x - m) * c);
        return exp2_fast(d) * fmaf(k1, d, k0);
    }
};
template <class F>
__device__ __forceinline__ float4 quad_of(float4 v, F f) {
    const Pair a = f(pair_of(v.x, v.y)), b = f(pair_of(v.z, v.w));
    return make_float4(low_of(a), high_of(a), low_of(b), high_of(b));
}
template <int THREADS, class F>
__device__ __forceinline__ void write_part(const Part& part, int q, float* g, float4 (&v)[kQuads], float loose, bool none, F f) {
    const bool vec = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(part.p)) & 15) == 0;
    float4 next[kQuads];
#pragma unroll 1
    for (int t = 0; t < q; t += THREADS) {
        if (t + THREADS < q) load_step(part, q, t + THREADS, next);
#pragma unroll
        for (int u = 0; u < kQuads; ++u) {
            const int i = u * q + t + (int)threadIdx.x;
            if (i >= part.n4) continue;
            float* to = g + part.head + 4 * i;
            const float4 o = none ? make_float4(0.f, 0.f, 0.f, 0.f) : quad_of(v[u], f);
            if (vec) *reinterpret_cast<float4*>(to) = o;
            else { to[0] = o.x; to[1] = o.y; to[2] = o.z; to[3] = o.w; }
        }
#pragma unroll
        for (int u = 0; u < kQuads; ++u) v[u] = next[u];
    }
    if ((int)threadIdx.x < part.n - 4 * part.n4) g[part.loose(threadIdx.x)] = none ? 0.0f : f(loose);
}

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
    unsigned long long best[kMaxList];     // largest first
    float4 hit[kHits];                     // quads, and their numbers
    int hit_at[kHits];
    uint32_t bound[2][kRowWarps];
    int n_hits[2], n_list[2], scanned[kRowWarps];
};
// behind it, where a row has a cluster: the best of all its CTAs, kMaxList places each, in the first one

// A bound that at least k of the threads' values reach: every warp's r-th largest, r = k / warps rounded up, and of those the smallest.
// All threads; one barrier inside; calls alternate between the two `bound`s.
__device__ __forceinline__ uint32_t bound_of(uint32_t mine, int k, uint32_t* bound) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t top = 0;
#pragma unroll 1
    for (int r = (k + kRowWarps - 1) / kRowWarps; r > 0; --r) {
        top = __reduce_max_sync(0xffffffffu, mine);
        const unsigned at = __ballot_sync(0xffffffffu, mine == top);
        if (lane == __ffs(at) - 1) mine = 0;
    }
    if (lane == 0) bound[warp] = top;
    __syncthreads();
    return __reduce_min_sync(0xffffffffu, bound[lane & (kRowWarps - 1)]);
}
// f(rank, candidate) for the k largest of list[0 .. n).  No two candidates are equal: their places differ.  The fewer they are, the more lanes
// count for one of them.
template <class F>
__device__ __forceinline__ void each_best(const unsigned long long* list, int n, int k, F f) {
    const int log = n <= 32 ? 3 : n <= 64 ? 2 : n <= 128 ? 1 : 0, lanes = 1 << log;
    const int part = threadIdx.x & (lanes - 1);
#pragma unroll 1
    for (int first = 0; first < n; first += kRowThreads >> log) {
        const int i = first + (threadIdx.x >> log);
        if (first + (((int)threadIdx.x & ~31) >> log) >= n) break;           // the whole warp
        const unsigned long long v = list[min(i, n - 1)];
        int rank = 0, j = part;
#pragma unroll 1
        for (; j + 3 * lanes < n; j += 4 * lanes) {
            unsigned long long w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = list[j + u * lanes];
#pragma unroll
            for (int u = 0; u < 4; ++u) rank += w[u] > v;
        }
#pragma unroll 1
        for (; j < n; j += lanes) rank += list[j] > v;
#pragma unroll 1
        for (int o = 1; o < lanes; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if (part == 0 && i < n && rank < k) f(rank, v);
    }
}
// f(rank, candidate) for the k largest of `lists` ordered lists, kMaxList places apart, 0 behind their ends: in each, those in front of a candidate
// are found by halving, in all lists at once.
template <class F>
__device__ __forceinline__ void each_best_of(const unsigned long long* list, int lists, int k, F f) {
    const int first = 1 << (31 - __clz(k));
#pragma unroll 1
    for (int i = threadIdx.x; i < lists * k; i += kRowThreads) {
        const int own = i / k, at = i - own * k;
        const unsigned long long v = list[own * kMaxList + at];
        int rank[kMaxCluster] = {};
#pragma unroll 1
        for (int half = first; half > 0; half >>= 1) {
            unsigned long long w[kMaxCluster];
#pragma unroll
            for (int o = 0; o < kMaxCluster; ++o) w[o] = o < lists && rank[o] + half <= k ? list[o * kMaxList + rank[o] + half - 1] : 0ull;
#pragma unroll
            for (int o = 0; o < kMaxCluster; ++o) rank[o] += w[o] > v ? half : 0;
        }
        int all = 0;
#pragma unroll
        for (int o = 0; o < kMaxCluster; ++o) all += rank[o];     // in its own list too: `at` are in front of it
        if (v != 0 && all < k) f(all, v);
    }
}
// To list: the values of a quad at `at` that reach `least`, or are above it (strict).
__device__ __forceinline__ void take(Selection& z, int* count, float4 v, int at, float least, bool strict) {
    const float w[4] = {v.x, v.y, v.z, v.w};
    unsigned which = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) which |= (strict ? w[i] > least : w[i] >= least) ? 1u << i : 0u;
    if (which == 0) return;
    int to = atomicAdd(count, __popc(which));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (which >> i & 1u) { if (to < kCandidates) z.list[to] = candidate(w[i], at + i); ++to; }
}
__device__ __forceinline__ float4 alone(float v) { return make_float4(v, NAN, NAN, NAN); }       // as a quad of which nothing else is taken
// ... of a whole part, from memory.  All threads.
__device__ __noinline__ void take_part(Selection& z, int* count, const float* p, int n, int c0, float least, bool strict) {
    const Part part(p, n);
#pragma unroll 1
    for (int t = threadIdx.x; t < part.n4; t += kQuads * kRowThreads) {
        float4 v[kQuads];
#pragma unroll
        for (int u = 0; u < kQuads; ++u) v[u] = load_behind(part.quads() + min(t + u * kRowThreads, part.n4 - 1));
#pragma unroll
        for (int u = 0; u < kQuads; ++u)
            if (t + u * kRowThreads < part.n4) take(z, count, v[u], c0 + part.head + 4 * (t + u * kRowThreads), least, strict);
    }
    if ((int)threadIdx.x < part.n - 4 * part.n4) {
        const int at = part.loose(threadIdx.x);
        take(z, count, alone(load_behind(part.p + at)), c0 + at, least, strict);
    }
}
// The first of those equal to `least` to list[n .. k_part).
__device__ __noinline__ void fill_equal(Selection& z, const float* p, int part_n, int c0, float least, int n, int k_part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
    for (int c = 0; c < part_n && n < k_part; c += kRowThreads) {
        const int at = c + threadIdx.x;
        const bool hit = at < part_n && load_behind(p + at) == least;
        const unsigned hits = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) z.scanned[warp] = __popc(hits);
        __syncthreads();
        int before = n, all = n;
        for (int w = 0; w < kRowWarps; ++w) { if (w < warp) before += z.scanned[w]; all += z.scanned[w]; }
        before += __popc(hits & ((1u << lane) - 1));
        if (hit && before < k_part) z.list[before] = candidate(least, c0 + at);
        n = min(all, k_part);
        __syncthreads();
    }
}
// Many equal values, or many large ones in few threads: the values above `least` alone, and the first of those equal to it where they are too few;
// while there is no room for them, the k-th largest of those that there is room for becomes `least` (k of the part reach it, and each of them is
// above the old one).  At least k_part of the part reach `least`.  Returns their number.
__device__ __noinline__ int take_few(Selection& z, int* count, const float* p, int part_n, int c0, float least, int k, int k_part) {
#pragma unroll 1
    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) *count = 0;
        __syncthreads();
        take_part(z, count, p, part_n, c0, least, true);
        __syncthreads();
        const int n = *count;
        if (n <= kCandidates) {
            if (n < k_part) fill_equal(z, p, part_n, c0, least, n, k_part);
            return max(n, k_part);
        }
        each_best(z.list, kCandidates, k, [&](int rank, unsigned long long v) { if (rank == k - 1) z.best[0] = v; });
        __syncthreads();
        least = unordered((uint32_t)(z.best[0] >> 32));
    }
}

// ---- what a row's CTAs share -------------------------------------------------------------------------------------------
struct RowShared {
    float wm[2][kRowWarps], ws[2][kRowWarps], wa[2][kRowWarps];    // of this row and of the one before, which may still be read
    float cm[2][kMaxCluster], cs[2][kMaxCluster], ca[2][kMaxCluster];       // written by the cluster's CTAs
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
    int n_top, last_bound;             // the last step behind which a bound is taken
    float* row_stats;
    const int* teacher_ids;
    const float* teacher_logits;
    int n_teacher;
    float* losses;
    const float* grad_out;             // with grad_logits
    float per_row;                     // 1 / (T rows)
    float* grad_logits;
    int* err_word;                     // where a bounded wait gives up
};

// ---- a teacher's lists, by one warp -----------------------------------------------------------------------------------
// It goes ahead of the others: the ids and logits of the item after the next and the student's logits at the ids of the next are on their way
// (asynchronous copies; a loop of loads would wait for each) while it works on the lists before.
struct __align__(16) TeacherList {
    int id[kMaxList];                  // outside [0, cols): no entry
    float t[kMaxList], log_t[kMaxList], x[kMaxList];                // probabilities, their logarithms, the student's logits
    float g[kMaxList];                 // the gradients at the entries (ring)
    float sum;                         // of the exponentials; 0: an empty list
    bool twice;                        // a token is named more than once
};
template <class P>
__device__ __forceinline__ void list_fetch(TeacherList& l, const P& p, size_t row) {
    const size_t at = row * (size_t)p.n_teacher;
    for (int i = threadIdx.x & 31; i < p.n_teacher; i += 32) {
        copy_async4(&l.id[i], p.teacher_ids + at + i);
        copy_async4(&l.t[i], p.teacher_logits + at + i);
    }
}
template <class P>
__device__ __forceinline__ void list_gather(TeacherList& l, const P& p, size_t row) {
    const float* x = p.logits + row * p.stride;
    for (int i = threadIdx.x & 31; i < p.n_teacher; i += 32) {
        const int id = l.id[i];
        if (id >= 0 && id < p.cols) copy_async4(&l.x[i], x + id);
        else l.t[i] = -INFINITY;
    }
}
// Probabilities t = exp2((a - top) c) / sum of the logits a, and their logarithms, which only a loss needs.
template <class P>
__device__ __forceinline__ void list_terms(TeacherList& l, const P& p) {
    const int lane = threadIdx.x & 31;
    float top = -FLT_MAX, sum = 0.0f;
    for (int i = lane; i < p.n_teacher; i += 32) top = fmaxf(top, l.t[i]);
    top = warp_top(top);
    for (int i = lane; i < p.n_teacher; i += 32) {
        const float d = l.t[i] - top, e = exp2_fast(clamp_low(d * p.c));
        l.log_t[i] = d;
        l.t[i] = e;
        sum += e;
    }
    sum = warp_add(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, log_sum = logf(sum);
    for (int i = lane; i < p.n_teacher; i += 32) { l.t[i] *= inv; l.log_t[i] = l.log_t[i] * p.inv_t - log_sum; }
    if (lane == 0) l.sum = sum;
    __syncwarp();
}
template <class F>
__device__ __forceinline__ float list_loss(const TeacherList& l, int n, F log_prob) {
    float loss = 0.0f;
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const float t = l.t[i];
        if (t != 0.0f) loss += t * (l.log_t[i] - log_prob(l.x[i]));
    }
    return warp_add(loss);
}
// Whether two entries of a list name the same token.  All lanes take part in every step: what a lane has found keeps it from none.
template <class P>
__device__ __forceinline__ bool list_twice(const TeacherList& l, const P& p) {
    const int lane = threadIdx.x & 31;
    bool twice = false;
#pragma unroll 1
    for (int i = 0; i < p.n_teacher; i += 32) {
        const int id = i + lane < p.n_teacher ? l.id[i + lane] : -1;
        const bool entry = id >= 0 && id < p.cols;
        const unsigned same = __match_any_sync(0xffffffffu, entry ? id : -1 - lane);
        twice |= entry && same != 1u << lane;
#pragma unroll 1
        for (int j = i + 32; j < p.n_teacher; j += 4) {           // against each entry of the groups of 32 behind it
            const int4 other = *reinterpret_cast<const int4*>(&l.id[j]);
            const bool found = id == other.x || (id == other.y && j + 1 < p.n_teacher) || (id == other.z && j + 2 < p.n_teacher) || (id == other.w && j + 3 < p.n_teacher);
            twice |= entry && found;
        }
    }
    return __any_sync(0xffffffffu, twice);
}
// The gradients of the listed tokens in [c0, c0 + cn), behind the rest of g: f(entry, place) for the first entry that names a token, and the
// probabilities of all its entries, in their order, to be taken off.
template <class F>
__device__ __forceinline__ void each_listed(const TeacherList& l, int n, int c0, int cn, F f) {
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const int id = l.id[i];
        if (id < c0 || id - c0 >= cn) continue;
        float t = l.t[i];
        if (l.twice) {
            bool first = true;
            t = 0.0f;
            for (int j = 0; j < n; ++j)
                if (l.id[j] == id) { t += l.t[j]; first = first && j >= i; }
            if (!first) continue;
        }
        f(i, id - c0, t);
    }
}
// The same at every entry, from the student's logits: entries that name the same token get the same.
template <class F>
__device__ __forceinline__ void list_gradients(TeacherList& l, int n, float up, F value) {
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        float t = l.t[i];
        if (l.twice) {
            t = 0.0f;
            for (int j = 0; j < n; ++j)
                if (l.id[j] == l.id[i]) t += l.t[j];
        }
        l.g[i] = value(l.x[i]) - t * up;
    }
}
// From the student's logits:
template <class F>
__device__ __forceinline__ void list_write(const TeacherList& l, int n, float* g, int c0, int cn, float up, F value) {
    each_listed(l, n, c0, cn, [&](int i, int at, float t) { g[at] = value(l.x[i]) - t * up; });
}
// The lists of items 0, 1, ... of a CTA: row(i) is an item's row.
template <int LISTS, class P, class R>
struct ListWarp {
    TeacherList* lists;                // LISTS of them, three or more
    const P& p;
    size_t items;                      // of this CTA
    R row;
    __device__ __forceinline__ TeacherList& of(size_t i) { return lists[i % LISTS]; }
    // before the first item
    __device__ __forceinline__ void start() {
        if (items == 0) return;
        list_fetch(of(0), p, row(0));
        if (items > 1) list_fetch(of(1), p, row(1));
        copies_end();
        copies_wait<0>();
        __syncwarp();
        list_gather(of(0), p, row(0));
        copies_end();
        __syncwarp();
        list_terms(of(0), p);
        const bool twice = list_twice(of(0), p);
        if ((threadIdx.x & 31) == 0) of(0).twice = twice;
        copies_wait<0>();
        __syncwarp();
    }
    // while item i is at work and all of item i - 1 is done: the next one's terms and student logits
    __device__ __forceinline__ void ahead(size_t i) {
        copies_wait<0>();
        __syncwarp();
        if (i + 1 < items) list_gather(of(i + 1), p, row(i + 1));
        if (i + 2 < items) list_fetch(of(i + 2), p, row(i + 2));
        copies_end();
        __syncwarp();
        if (i + 1 < items) {
            list_terms(of(i + 1), p);
            const bool twice = list_twice(of(i + 1), p);
            if ((threadIdx.x & 31) == 0) of(i + 1).twice = twice;
        }
    }
    // before an item's student logits are used
    __device__ __forceinline__ void arrived() {
        copies_wait<0>();
        __syncwarp();
    }
};

// The statistics that the backward call takes: no sum where the row has no entries, none that is a number where its list is none.
__device__ __forceinline__ float gradient_sum(float s, float list_sum) { return list_sum == 0.0f ? 0.0f : list_sum == list_sum ? s : list_sum; }
__device__ __forceinline__ void list_result(const VocabRows& p, const TeacherList& l, size_t row, float m, float s, float loss) {
    if ((threadIdx.x & 31) != 0) return;
    p.losses[row] = loss;
    if (p.row_stats != nullptr) { p.row_stats[2 * row] = m; p.row_stats[2 * row + 1] = gradient_sum(s, l.sum); }
}

// One row at a time on a CTA, or a row on a cluster's CTAs where there are few.
// TOP: a thread's first step is a sample of the row; the quads with something above the bound that it gives are noted as the row goes by, and
// looked at again under the bound of all that the threads have seen.
// That stays behind 1 % of the values of a long row and costs no second look at memory: 30 us of 110, which are issue slots (71 % of them
// busy), the barriers of a row and 36 bytes a thread that 64 registers do not hold (lists: 8, with the gradient 204).  Where more than kHits quads are noted (lists of 128 of long rows) the row is read again.
// LIST, GRAD: the last warp has the teacher's lists and forms the losses.  GRAD: the row goes by a second time (out of L2, where rows are few or short; long
// ones go through the ring below), becomes its gradient, and that warp writes the listed tokens' gradients while the next row is at work.
enum RowWork { kPlain, kTop, kList, kGrad };
template <bool ENTROPY, RowWork WORK>
__global__ void __launch_bounds__(kRowThreads, 4) vocab_rows_kernel(VocabRows p) {
    constexpr bool TOP = WORK == kTop, DISTILL = WORK == kList || WORK == kGrad, GRAD = WORK == kGrad;
    constexpr int THREADS = kRowThreads - (DISTILL ? 32 : 0), WARPS = THREADS / 32;       // that work on rows
    grid_release();
    extern __shared__ __align__(16) unsigned char dynamic[];
    Selection& z = *reinterpret_cast<Selection*>(dynamic + kStreamBytes);       // TOP
    unsigned long long* gathered = reinterpret_cast<unsigned long long*>(dynamic + kStreamBytes + sizeof(Selection));
    TeacherList* lists = reinterpret_cast<TeacherList*>(dynamic + kStreamBytes);                   // DISTILL
    __shared__ RowShared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ranks = p.cluster, rank = ranks > 1 ? (int)(blockIdx.x % ranks) : 0;
    const int per = ((p.cols + ranks - 1) / ranks + 3) & ~3;
    const int c0 = min(p.cols, rank * per), cn = min(p.cols, c0 + per) - c0;
    const size_t first = blockIdx.x / ranks, step = gridDim.x / ranks, mine = (p.rows - first + step - 1) / step;
    const int k = p.n_top, k_part = min(k, cn);
    if (ranks > 1) { cluster_arrive(); cluster_wait(); }          // every CTA of the cluster runs
    if (TOP && threadIdx.x == 0) z.n_hits[0] = z.n_hits[1] = z.n_list[0] = z.n_list[1] = 0;
    if (DISTILL && threadIdx.x == 0)                              // the one that joins statistics of WARPS takes a power of two of them
        for (int w = WARPS; w < kRowWarps; ++w) { sh.wm[0][w] = sh.wm[1][w] = -FLT_MAX; sh.ws[0][w] = sh.ws[1][w] = 0.0f; }
    grid_wait();
    const bool of_lists = DISTILL && warp == WARPS;
    auto row_of = [&](size_t i) { return first + i * step; };
    auto part_of = [&](size_t i) { return Part(p.logits + row_of(i) * p.stride + c0, cn); };
    ListWarp<3, VocabRows, decltype(row_of)> list_warp = {lists, p, mine, row_of};
    if (of_lists) list_warp.start();
    Stream<THREADS, decltype(part_of)> stream(dynamic, part_of, of_lists ? 0 : mine, cn);
    const int q = stream.q;
    const float up = GRAD ? load_behind(p.grad_out) * p.per_row : 0.0f;
    // GRAD, of the row before too, whose listed tokens are written when all of its gradient is
    float gm = 0.0f, gf = 0.0f;
    bool none = true;
    auto write_behind = [&](size_t item) {
        if (!none)
            list_write(list_warp.of(item), p.n_teacher, p.grad_logits + row_of(item) * p.stride + c0, c0, cn, up, ProbGrad{gm, p.c, gf});
    };
    for (size_t item = 0; item < mine; ++item) {
        const size_t row = row_of(item);
        const int turn = (int)(item & 1);
        const float* x = p.logits + row * p.stride;
        const Part part(x + c0, cn);
        Running<ENTROPY> run;
        float over = INFINITY, least = -INFINITY, x_token = 0.0f, loose = -INFINITY;
        int token = -1;
        const bool has_loose = (int)threadIdx.x < part.n - 4 * part.n4;
        float4 again[kQuads];                                     // GRAD: the first step a second time
        if (!of_lists) {
            if (has_loose) loose = load_behind(part.p + part.loose(threadIdx.x));
            if (!DISTILL && p.tokens != nullptr && threadIdx.x == kResultThread && rank == 0) {
                token = load_behind(p.tokens + row);
                if (token < 0 || token >= p.cols) token = -1;
                else x_token = load_behind(x + token);
            }
#pragma unroll 1
            for (int t = 0; t < q; t += THREADS) {
                float4 v[kQuads];
                stream.take(t, part.n4, v);
                float top = top_of(v[0]);
#pragma unroll
                for (int u = 1; u < kQuads; ++u) top = fmaxf(top, top_of(v[u]));
                run.quads(v, top, p.c);
                stream.next();
                if (TOP) {
                    if (q == THREADS) {                           // the sample is all
                        run.one(loose, p.c);
                        least = unordered(max(bound_of(ordered(run.largest()), k, z.bound[0]), ordered(-INFINITY)));
#pragma unroll
                        for (int u = 0; u < kQuads; ++u) {
                            const int i = u * q + (int)threadIdx.x;
                            if (i < part.n4) take(z, &z.n_list[turn], v[u], c0 + part.head + 4 * i, least, false);
                        }
                    } else {
                        const int past = t / THREADS;
                        if (past <= p.last_bound && (past & (past + 1)) == 0)
                            over = unordered(max(bound_of(ordered(run.largest()), k, z.bound[__popc(past) & 1]), ordered(-INFINITY)));
                        if (top > over) {
                            unsigned which = 0;
#pragma unroll
                            for (int u = 0; u < kQuads; ++u) which |= top_of(v[u]) > over ? 1u << u : 0u;
                            int at = atomicAdd(&z.n_hits[turn], __popc(which));
#pragma unroll
                            for (int u = 0; u < kQuads; ++u)
                                if (which >> u & 1u) {
                                    if (at < kHits) { z.hit[at] = v[u]; z.hit_at[at] = u * q + t + (int)threadIdx.x; }
                                    ++at;
                                }
                        }
                    }
                }
            }
            if (!TOP || q != THREADS) run.one(loose, p.c);
            if (GRAD) load_step(part, q, 0, again);
        }
        Stats<ENTROPY> st = run.sums();
        if (!of_lists) {
            st.template join<32>(p.c);
            if (lane == 0) { sh.wm[turn][warp] = st.m; sh.ws[turn][warp] = st.s; if (ENTROPY) sh.wa[turn][warp] = st.a; }
        }
        if (TOP) {
            int* count = &z.n_list[turn];
            if (q != THREADS) {
                const int bounds = 32 - __clz(min(q / THREADS, p.last_bound + 1));       // taken on the way
                least = unordered(max(bound_of(ordered(run.largest()), k, z.bound[bounds & 1]), ordered(-INFINITY)));
                const int hits = z.n_hits[turn];
                const bool strict = q > 0 && !(least > over);     // among the quads that were not noted some may equal it
                if (hits > kHits) take_part(z, count, part.p, part.n, c0, least, false);
                else {
#pragma unroll 1
                    for (int i = threadIdx.x; i < hits; i += kRowThreads) take(z, count, z.hit[i], c0 + part.head + 4 * z.hit_at[i], least, strict);
                    if (has_loose) take(z, count, alone(loose), c0 + part.loose(threadIdx.x), least, strict);
                }
            } else if (has_loose) take(z, count, alone(loose), c0 + part.loose(threadIdx.x), least, false);
        }
        if (of_lists) list_warp.arrived();                        // before anything of this row may become its gradient (grad_logits == logits)
        __syncthreads();                                          // GRAD: and all of the gradient of the row before is there
        if (GRAD && of_lists && item > 0) write_behind(item - 1);
        st.m = sh.wm[turn][lane & (kRowWarps - 1)];
        st.s = sh.ws[turn][lane & (kRowWarps - 1)];
        if (ENTROPY) st.a = sh.wa[turn][lane & (kRowWarps - 1)];
        st.template join<kRowWarps>(p.c);
        int n = 0;
        if (TOP) {
            n = z.n_list[turn];
            if (threadIdx.x == 0) z.n_hits[turn ^ 1] = z.n_list[turn ^ 1] = 0;       // for the next row
            if (!(st.s == st.s)) n = 0;                           // not a number: its places are not looked at
            else if (n > kCandidates || n < k_part) n = take_few(z, &z.n_list[turn], part.p, part.n, c0, least, k, k_part);
        }
        if (ranks > 1) {
            // the first CTA gets all statistics and every part's best
            if (TOP) {
                each_best(z.list, n, k_part, [&](int r, unsigned long long c) { z.best[r] = c; });
                __syncthreads();
                if ((int)threadIdx.x < k)
                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_address(&gathered[rank * kMaxList + threadIdx.x], 0)),
                                 "l"((int)threadIdx.x < min(n, k_part) ? z.best[threadIdx.x] : 0ull) : "memory");       // 0: below every candidate
            }
            if ((int)threadIdx.x < (GRAD ? ranks : 1)) {          // GRAD: all of them
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(&sh.cm[turn][rank], threadIdx.x)), "f"(st.m) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(&sh.cs[turn][rank], threadIdx.x)), "f"(st.s) : "memory");
                if (ENTROPY) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(&sh.ca[turn][rank], threadIdx.x)), "f"(st.a) : "memory");
            }
            cluster_arrive();
            cluster_wait();
            if (!GRAD && rank > 0) return;                        // a cluster has one row (launch_forward)
            Stats<ENTROPY> all;
            for (int r = 0; r < ranks; ++r) all.m = fmaxf(all.m, sh.cm[turn][r]);
            for (int r = 0; r < ranks; ++r) {
                Stats<ENTROPY> one;
                one.m = sh.cm[turn][r]; one.s = sh.cs[turn][r];
                if (ENTROPY) one.a = sh.ca[turn][r];
                one.raise(all.m, p.c);
                all.s += one.s; all.a += one.a;
            }
            st = all;
        }
        const float m = st.m, s = st.s, log_s = logf(s);
        auto log_prob = [&](float value) { return s == 0.0f ? -INFINITY : (value - m) * p.inv_t - log_s; };      // s == 0: nothing is left of the row
        if (!DISTILL && threadIdx.x == kResultThread) {
            if (p.row_stats != nullptr) { p.row_stats[2 * row] = m; p.row_stats[2 * row + 1] = s; }
            if (p.logprobs != nullptr) p.logprobs[row] = token < 0 ? 0.0f : log_prob(x_token);
            if (ENTROPY) p.entropy[row] = s == 0.0f ? 0.0f : log_s - st.a / s * kLn2;
        }
        if (TOP) {
            const size_t at = row * (size_t)k;
            if (!(s == s)) {
                if ((int)threadIdx.x < k) {
                    if (p.top_ids != nullptr) p.top_ids[at + threadIdx.x] = -1;
                    if (p.top_logprobs != nullptr) p.top_logprobs[at + threadIdx.x] = s;
                }
                continue;
            }
            auto put = [&](int r, unsigned long long c) {
                if (p.top_ids != nullptr) p.top_ids[at + r] = (int)(0xffffffffu - (uint32_t)c);
                if (p.top_logprobs != nullptr) p.top_logprobs[at + r] = log_prob(unordered((uint32_t)(c >> 32)));
            };
            if (ranks == 1) each_best(z.list, n, k, put);
            else each_best_of(gathered, ranks, k, put);
        }
        if (GRAD) {
            const float sg = gradient_sum(s, list_warp.of(item).sum);
            gm = m;
            gf = up / sg;
            none = sg == 0.0f || up == 0.0f;
        }
        if (of_lists) {
            const TeacherList& list = list_warp.of(item);
            const float loss = list_loss(list, p.n_teacher, log_prob);
            if (rank == 0) list_result(p, list, row, m, s, loss);
            list_warp.ahead(item);
        } else if (GRAD) write_part<THREADS>(part, q, p.grad_logits + row * p.stride + c0, again, loose, none, ProbGrad{m, p.c, gf});
    }
    if (GRAD) {
        __syncthreads();
        if (of_lists) write_behind(mine - 1);
    }
}

// ---- loss and gradient of long rows in one pass ---------------------------------------------------------------------------
// A row comes to shared memory once, in chunks by bulk copies, becomes its gradient there, and goes out by bulk copies: a ring of chunks in which the
// next rows come while this one is at work and the one before goes.  The threads themselves neither load nor store: behind their own stores all
// of an SM's memory instructions, those on shared memory among them, waited two thirds of the time.  Bound by memory, read and write.  4096 x 32000 with lists of
// 64: 184 us, 88 % of the copy's rate, 5000 x 20000 148 us (84 %), 1000 x 128256 222 us (72 %); the rows of 32000 a second time out of L2 300 us with four rows on an
// SM, of which L2 keeps none, 325 with three, 398 with two, 549 with one; a row in shared memory with the threads' own copies and stores 219.
// Two more warps: one has the teacher's lists, forms the losses and the listed tokens' gradients; one issues the copies and writes those gradients a row behind,
// when the bulk copies of their row are done.
// Nothing may be ahead of the copying warp by more than its ring: a row's statistics need all of its chunks, of which there are kRingAhead rows beside the one
// that goes out, so that while that is row i, rows up to i + 2 have statistics and lists up to row i + 4 are fetched; of row i - 1 the list is still needed.
constexpr int kRingThreads = 512;      // that work on rows
constexpr int kRingWarps = kRingThreads / 32;
constexpr size_t kRingBytes = 208 * 1024;
constexpr int kRingMost = 12;          // chunks of a row
constexpr int kRingAhead = 2;          // rows in the ring beside the one that goes out, at most
constexpr int kRingSlots = (kRingAhead + 1) * kRingMost;
constexpr int kRingLists = 4 + kRingAhead;                        // from the row before the one that goes out to two behind the last one in the ring
constexpr int kRingErr = 61;
struct Ring {
    int chunk, chunks, slots;          // quads of a chunk, chunks of a row, chunks of the ring
};
__device__ __forceinline__ void bulk_load(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_store(void* to, uint32_t from, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_end() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// To the CTA `rank` of the cluster: a pair of values, counted by the barrier there.
__device__ __forceinline__ void send_pair(const void* to, const void* bar, int rank, float a, float b) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(cluster_address(to, rank)), "f"(a), "f"(b),
                 "r"(cluster_address(bar, rank)) : "memory");
}
// A completed phase once more, for what other CTAs have written.
__device__ __forceinline__ void cluster_acquire(uint32_t bar, uint32_t parity) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%0], %1;\n\t}" ::"r"(bar), "r"(parity) : "memory");
}
// CLUSTER: a CTA has a part of a row; the parts' statistics cross the cluster once a row, to barriers that count them.
template <bool CLUSTER>
__global__ void __launch_bounds__(kRingThreads + 64, 1) distill_ring_kernel(VocabRows p, Ring r) {
    grid_release();
    extern __shared__ __align__(16) unsigned char dynamic[];
    float4* ring = reinterpret_cast<float4*>(dynamic);
    __shared__ float wm[2][kRingWarps], ws[2][kRingWarps];
    __shared__ bool stat_none[4];
    __shared__ TeacherList lists[kRingLists];
    __shared__ __align__(8) unsigned long long full[kRingSlots], done[kRingSlots];
    __shared__ __align__(8) float2 parts[2][kMaxCluster];
    __shared__ __align__(8) unsigned long long crossed[2];
    __shared__ int gave_up;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ranks = CLUSTER ? p.cluster : 1, rank = CLUSTER ? (int)(blockIdx.x % ranks) : 0;
    const int per = ((p.cols + ranks - 1) / ranks + 3) & ~3;
    const int c0 = rank * per, cn = min(p.cols, c0 + per) - c0;
    const size_t first = blockIdx.x / ranks, step = gridDim.x / ranks, mine = (p.rows - first + step - 1) / step;
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int b = 0; b < r.slots; ++b) { mbar_init(smem_u32(&full[b]), 1); mbar_init(smem_u32(&done[b]), kRingWarps + 1); }
        for (int b = 0; b < 2; ++b) mbar_init(smem_u32(&crossed[b]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (CLUSTER) { cluster_arrive(); cluster_wait(); }            // the others' barriers are there
    grid_wait();
    auto row_of = [&](size_t i) { return first + i * step; };
    auto part_of = [&](size_t i) { return Part(p.logits + row_of(i) * p.stride + c0, cn); };
    ListWarp<kRingLists, VocabRows, decltype(row_of)> list_warp = {lists, p, mine, row_of};
    const float up = load_behind(p.grad_out) * p.per_row;
    // Where a wait runs out the call's results are void: the error word says so, nobody waits any more, and every loop runs to its end.
    auto gone = [&] {
        if (lane == 0) {
            gave_up = 1;
            *p.err_word = kRingErr;
        }
        __syncwarp();
    };
    if (warp == kRingWarps + 1) {
        auto quads_of = [&](const Part& part, int c) { return max(0, min(r.chunk, part.n4 - c * r.chunk)); };
        size_t ahead_item = 0;                                    // next to load: its chunk ahead_c
        int ahead_c = 0, slot_in = 0, slot_out = 0;
        Part ahead = part_of(0);
        auto load = [&] {                                         // one lane
            if (ahead_item >= mine) return;
            const uint32_t n = quads_of(ahead, ahead_c) * 16u, bar = smem_u32(&full[slot_in]);
            mbar_expect_tx(bar, n);
            if (n > 0) bulk_load(smem_u32(ring + slot_in * r.chunk), ahead.quads() + ahead_c * r.chunk, n, bar);
            if (++ahead_c == r.chunks) {
                ahead_c = 0;
                if (++ahead_item < mine) ahead = part_of(ahead_item);
            }
            if (++slot_in == r.slots) slot_in = 0;
        };
        if (lane == 0)
            for (int i = 0; i < r.slots - 1; ++i) load();
        __syncwarp();
        uint32_t parity = 0;
        bool ok = true;
        auto write_behind = [&](size_t item) {
            if (!ok || stat_none[item & 3]) return;
            const TeacherList& list = list_warp.of(item);
            float* g = p.grad_logits + row_of(item) * p.stride + c0;
            for (int i = lane; i < p.n_teacher; i += 32) {
                const int id = list.id[i];
                if (id >= c0 && id - c0 < cn) g[id - c0] = list.g[i];
            }
        };
        for (size_t item = 0; item < mine; ++item) {
            const Part part = part_of(item);
            float* g = p.grad_logits + row_of(item) * p.stride + c0 + part.head;
#pragma unroll 1
            for (int c = 0; c < r.chunks; ++c) {
                if (ok && !mbar_wait_warp(smem_u32(&done[slot_out]), parity, &gave_up)) { ok = false; gone(); }
                if (lane == 0 && ok) {
                    const int n = quads_of(part, c);
                    if (n > 0) bulk_store(g + 4 * c * r.chunk, smem_u32(ring + slot_out * r.chunk), n * 16u);
                    bulk_end();
                    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    load();                                       // to where the chunk before this one was
                }
                if (++slot_out == r.slots) { slot_out = 0; parity ^= 1u; }
            }
            // what is pending then is of this row
            if (lane == 0) {
                if (r.chunks == 1) asm volatile("cp.async.bulk.wait_group 1;" ::: "memory");
                else if (r.chunks == 2) asm volatile("cp.async.bulk.wait_group 2;" ::: "memory");
                else if (r.chunks < 7) asm volatile("cp.async.bulk.wait_group 3;" ::: "memory");
                else asm volatile("cp.async.bulk.wait_group 7;" ::: "memory");
            }
            __syncwarp();
            if (item > 0) write_behind(item - 1);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
        write_behind(mine - 1);
        if (*(volatile int*)&gave_up) {
            // loads that are still in flight land before the shared memory is released
            const unsigned long long t0 = clock64();
            while (clock64() - t0 < 2000000ull) {}
        }
        if (CLUSTER) { __syncwarp(); cluster_arrive(); cluster_wait(); }
        return;
    }
    const bool of_lists = warp == kRingWarps;
    if (of_lists) list_warp.start();
    int slot = 0;                                                 // of this row's first chunk
    uint32_t parity = 0;
    bool ok = true;
    for (size_t item = 0; item < mine; ++item) {
        const size_t row = row_of(item);
        const int turn = (int)(item & 1);
        const Part part = part_of(item);
        const bool has_loose = (int)threadIdx.x < part.n - 4 * part.n4;
        const float loose = has_loose ? load_behind(part.p + part.loose(threadIdx.x)) : -INFINITY;
        Running<false> run;
        int at_slot = slot;
        uint32_t at_parity = parity;
        if (!of_lists) {
#pragma unroll 1
            for (int c = 0; c < r.chunks; ++c) {
                if (ok && !mbar_wait_warp(smem_u32(&full[at_slot]), at_parity, &gave_up)) { ok = false; gone(); }
                const int n = min(r.chunk, part.n4 - c * r.chunk);
                const float4* chunk = ring + at_slot * r.chunk;
#pragma unroll 1
                for (int i = threadIdx.x; i < n; i += 4 * kRingThreads) {
                    float4 v[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        v[u] = i + u * kRingThreads < n ? chunk[i + u * kRingThreads] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    run.quads(v, fmaxf(fmaxf(top_of(v[0]), top_of(v[1])), fmaxf(top_of(v[2]), top_of(v[3]))), p.c);
                }
                if (++at_slot == r.slots) { at_slot = 0; at_parity ^= 1u; }
            }
            run.one(loose, p.c);
        }
        Stats<false> st = run.sums();
        if (!of_lists) {
            st.join<32>(p.c);
            if (lane == 0) { wm[turn][warp] = st.m; ws[turn][warp] = st.s; }
        }
        if (of_lists) list_warp.arrived();                        // before anything of this row may become its gradient (grad_logits == logits)
        asm volatile("bar.sync 1, %0;" ::"n"(kRingThreads + 32) : "memory");
        st.m = wm[turn][lane & (kRingWarps - 1)];
        st.s = ws[turn][lane & (kRingWarps - 1)];
        st.join<kRingWarps>(p.c);
        if (CLUSTER) {
            if (warp == 0) {
                if (lane == 0) mbar_expect_tx(smem_u32(&crossed[turn]), ranks * 8);
                if (lane < ranks) send_pair(&parts[turn][rank], &crossed[turn], lane, st.m, st.s);
            }
            const uint32_t phase = (uint32_t)(item >> 1) & 1u;
            if (ok && !mbar_wait_warp(smem_u32(&crossed[turn]), phase, &gave_up)) { ok = false; gone(); }
            if (ok) cluster_acquire(smem_u32(&crossed[turn]), phase);
            st = Stats<false>();
            if (lane < ranks) { st.m = parts[turn][lane].x; st.s = parts[turn][lane].y; }
            st.join<kMaxCluster>(p.c);
            st.m = __shfl_sync(0xffffffffu, st.m, 0);
            st.s = __shfl_sync(0xffffffffu, st.s, 0);
        }
        // an empty list or an empty row has no gradient, nor has a loss of which none is asked; a list that is not a number has none that is one
        const TeacherList& list = list_warp.of(item);
        const float m = st.m, s = st.s, sg = gradient_sum(s, list.sum);
        const bool none = sg == 0.0f || up == 0.0f;
        const float f = none ? 0.0f : up / sg;                    // 0 too where it underflows: the listed tokens' gradients may not
        if (of_lists) {
            if (!none) list_gradients(list_warp.of(item), p.n_teacher, up, ProbGrad{m, p.c, f});
            __syncwarp();
            if (lane == 0)
                for (int c = 0; c < r.chunks; ++c) {
                    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&done[slot])) : "memory");
                    if (++slot == r.slots) slot = 0;
                }
            const float log_s = logf(s);
            const float loss = list_loss(list, p.n_teacher, [&](float v) { return s == 0.0f ? -INFINITY : (v - m) * p.inv_t - log_s; });
            if (rank == 0) list_result(p, list, row, m, s, loss);
            list_warp.ahead(item);
            continue;
        }
        if (threadIdx.x == 0) stat_none[item & 3] = none;
        const ProbGrad value = {m, p.c, f};
        if (has_loose) p.grad_logits[row * p.stride + c0 + part.loose(threadIdx.x)] = none ? 0.0f : value(loose);
#pragma unroll 1
        for (int c = 0; c < r.chunks; ++c) {
            const int n = min(r.chunk, part.n4 - c * r.chunk);
            float4* chunk = ring + slot * r.chunk;
#pragma unroll 4
            for (int i = threadIdx.x; i < n; i += kRingThreads) chunk[i] = none ? make_float4(0.f, 0.f, 0.f, 0.f) : quad_of(chunk[i], value);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&done[slot])) : "memory");
            if (++slot == r.slots) { slot = 0; parity ^= 1u; }
        }
    }
    if (CLUSTER) { __syncwarp(); cluster_arrive(); cluster_wait(); }      // nothing more comes to this CTA's shared memory
}

// ---- gradients from kept statistics ------------------------------------------------------------------------------------
struct VocabGrad {
    const float* logits;
    size_t rows, stride;
    int cols, tiles, per;              // tiles of a row, their length
    float c, inv_t;                    // of lists: 1 / (T rows)
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

// What a row's gradient is formed from.
struct Terms {
    float k0, k1, up;
    int token;                         // -1: none
    bool none;                         // all of the gradient is 0
};
template <bool DISTILL>
__device__ __forceinline__ Terms grad_terms(const VocabGrad& p, size_t row, float m, float s) {
    Terms t = {0.0f, 0.0f, 0.0f, -1, s == 0.0f};
    if (DISTILL) {
        t.up = load_behind(p.grad_out) * p.inv_t;
        t.none = t.none || t.up == 0.0f;
        t.k0 = t.up / s;
        return t;
    }
    float h = 0.0f, H = 0.0f;
    if (p.grad_logprobs != nullptr) {
        t.token = load_behind(p.tokens + row);
        if (t.token < 0 || t.token >= p.cols) t.token = -1;
        else t.up = load_behind(p.grad_logprobs + row) * p.inv_t;
    }
    if (p.grad_entropy != nullptr) { h = load_behind(p.grad_entropy + row) * p.inv_t; H = load_behind(p.entropy + row); }
    t.none = t.none || (t.up == 0.0f && h == 0.0f);
    t.k0 = -(t.up + (h == 0.0f ? 0.0f : h * (H - logf(s)))) / s;
    t.k1 = -h * kLn2 / s;
    return t;
}

// dx_c = e_c (k0 + k1 d_c) + (what the named tokens add), with e_c = 2^((x_c - m) c): p_c enters through 1 / s in k0 and k1.
// Bound by memory, read and write: 4096 x 32000 in 161 us, a copy's rate; from lists of 64 176 us, as a CTA's writing ends in one warp's work.
// DISTILL: the first warp has an item's list on its way from the start, and takes the listed tokens' probabilities off when the rest is written.
template <bool DISTILL>
__global__ void __launch_bounds__(kRowThreads, 4) vocab_grad_kernel(VocabGrad p) {
    grid_release();
    grid_wait();
    __shared__ TeacherList list;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t items = p.rows * (size_t)p.tiles;
    const int q = quarter_of(p.per, kRowThreads);
    for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
        const size_t row = item / p.tiles;
        const int c0 = (int)(item - row * p.tiles) * p.per, cn = min(p.cols - c0, p.per);
        const float* x = p.logits + row * p.stride;
        const Part part(x + c0, cn);
        float* g = p.grad_logits + row * p.stride + c0;
        float4 v[kQuads];
        load_step(part, q, 0, v);
        const float loose = (int)threadIdx.x < part.n - 4 * part.n4 ? load_behind(part.p + part.loose(threadIdx.x)) : 0.0f;
        const float m = load_behind(p.row_stats + 2 * row), s = load_behind(p.row_stats + 2 * row + 1);
        if (DISTILL && warp == 0) { list_fetch(list, p, row); copies_end(); }
        const Terms terms = grad_terms<DISTILL>(p, row, m, s);
        float x_token = 0.0f;
        if (!DISTILL) {
            if (threadIdx.x == 0 && terms.token >= 0) x_token = load_behind(x + terms.token);
            __syncthreads();        // the token's logit is read before any of the row is written (grad_logits may be logits); other tiles' are not used
        }
        const EntropyGrad with_entropy = {m, p.c, terms.k0, terms.k1};
        if (DISTILL) write_part<kRowThreads>(part, q, g, v, loose, terms.none, ProbGrad{m, p.c, terms.k0});
        else write_part<kRowThreads>(part, q, g, v, loose, terms.none, with_entropy);
        __syncthreads();
        if (!DISTILL && threadIdx.x == 0 && !terms.none && terms.token >= c0 && terms.token < c0 + cn) g[terms.token - c0] = with_entropy(x_token) + terms.up;
        if (DISTILL && warp == 0) {
            copies_wait<0>();                                     // whatever the row asks for: the next item's list comes to the same place
            __syncwarp();
            if (terms.none) continue;
            for (int i = lane; i < p.n_teacher; i += 32)
                if (list.id[i] < 0 || list.id[i] >= p.cols) list.t[i] = -INFINITY;
            list_terms(list, p);
            const bool twice = list_twice(list, p);
            if (lane == 0) list.twice = twice;
            __syncwarp();
            each_listed(list, p.n_teacher, c0, cn, [&](int, int at, float t) { g[at] -= t * terms.up; });      // p is there
            __syncwarp();                                         // before the next item's list comes
        }
    }
}

// ---- short rows: W warps for each, which hold it in registers ----------------------------------------------------------------
// Up to 128 W J logits, J quads a lane: a barrier a row at most, no exponential before the warp's largest logit is known, a second look that costs nothing, and as
// many rows of an SM on their way as registers hold.  What a CTA of the kernel above spends on a row beside its logits, 2.4 us, is more than short rows take.  By such
// CTAs / here: 11000 x 1000 statistics 47 / 11 us, their gradient 40 / 14, lists' loss 54 / 17, loss and gradient 83 / 27; 40000 x 2000: 167 / 54 (92 % of the copy's rate),
// 161 / 101 (98 %), 177 / 94, 318 / 118 (84 %); 11000 x 4096 44 / 40, 61 / 59, 63 / 56, 143 / 74.
template <int W, int J>
struct ShortRow {
    Part part;
    float4 v[J];
    float loose;                       // outside the quads: one of the first lanes each
    __device__ __forceinline__ ShortRow(const float* row, int n) : part(row, n), loose(-INFINITY) {
        const int t = threadIdx.x % (32 * W);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            v[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (t + 32 * W * j < part.n4) v[j] = load_behind(part.quads() + t + 32 * W * j);
        }
        if (t < part.n - 4 * part.n4) loose = load_behind(part.p + part.loose(t));
    }
    // of this warp's part
    template <bool ENTROPY>
    __device__ __forceinline__ Stats<ENTROPY> stats(float c) const {
        float top = fmaxf(-FLT_MAX, loose);
#pragma unroll
        for (int j = 0; j < J; ++j) top = fmaxf(top, top_of(v[j]));
        top = warp_top(top);
        Running<ENTROPY> run;
        run.m = top;
        run.minus_m = pair_of(-top, -top);
#pragma unroll
        for (int j = 0; j < J; ++j) { run.terms(pair_of(v[j].x, v[j].y), c); run.terms(pair_of(v[j].z, v[j].w), c); }
        run.terms(pair_of(loose, -INFINITY), c);
        Stats<ENTROPY> st = run.sums();
        st.s = warp_add(st.s);
        if (ENTROPY) st.a = warp_add(st.a);
        return st;
    }
    template <class F>
    __device__ __forceinline__ void write(float* g, bool none, F f) const {
        const int t = threadIdx.x % (32 * W);
        const bool vec = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(part.p)) & 15) == 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (t + 32 * W * j >= part.n4) continue;
            float* to = g + part.head + 4 * (t + 32 * W * j);
            const float4 o = none ? make_float4(0.f, 0.f, 0.f, 0.f) : quad_of(v[j], f);
            if (vec) *reinterpret_cast<float4*>(to) = o;
            else { to[0] = o.x; to[1] = o.y; to[2] = o.z; to[3] = o.w; }
        }
        if (t < part.n - 4 * part.n4) g[part.loose(t)] = none ? 0.0f : f(loose);
    }
};
// The k largest of a row that a warp has, k <= kMaxList and the row's length: f(rank, candidate).  A bound that at least k values reach: the k-th largest of the largest of
// four groups of every lane, found by halving; those that reach it go to `list`, kCandidates places, and are ordered by counting.
template <int J, class F>
__device__ __forceinline__ void short_tops(const ShortRow<1, J>& r, int k, unsigned long long* list, F f) {
    const int lane = threadIdx.x & 31, n4 = r.part.n4;
    const bool has_loose = lane < r.part.n - 4 * n4;
    // the largest t of [lo, hi) with count(t) >= k, or one with k <= count(t) <= most; count(lo) >= k > count(hi)
    auto halve = [&](uint32_t& lo, uint32_t hi, int most, auto count) {
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int n = (int)__reduce_add_sync(0xffffffffu, (unsigned)count(unordered(mid)));
            if (n < k) hi = mid;
            else {
                lo = mid;
                if (n <= most) return;
            }
        }
    };
    float top[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        top[g] = g == 0 ? r.loose : -INFINITY;
#pragma unroll
        for (int j = g; j < J; j += 4) top[g] = fmaxf(top[g], top_of(r.v[j]));
    }
    const uint32_t all = ordered(-INFINITY), high = __reduce_max_sync(0xffffffffu, ordered(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))));
    uint32_t bound = k == 1 ? high : all;
    if (k > 1) halve(bound, high + 1, k, [&](float t) { return (top[0] >= t) + (top[1] >= t) + (top[2] >= t) + (top[3] >= t); });
    auto reach = [&](float t) {                                   // how many of the lane's
        int n = has_loose && r.loose >= t;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (lane + 32 * j < n4) n += (r.v[j].x >= t) + (r.v[j].y >= t) + (r.v[j].z >= t) + (r.v[j].w >= t);
        return n;
    };
    float least = unordered(bound);
    int mine = reach(least), n = (int)__reduce_add_sync(0xffffffffu, (unsigned)mine);
    bool fill = false;
    if (n > max(k + 32, 96)) {                                    // counting takes n^2 steps, halving 10 to 32 looks at the row
        halve(bound, high + 1, k + 32, reach);
        least = unordered(bound);
        mine = reach(least);
        n = (int)__reduce_add_sync(0xffffffffu, (unsigned)mine);
        fill = n > kCandidates;                                   // that many are equal to it, and fewer than k above
    }
    // those that pass, to where the lanes in front of this one end
    auto put = [&](auto pass, int to) {
        auto one = [&](float v, int at) { if (pass(v)) { if (to < kCandidates) list[to] = candidate(v, at); ++to; } };
        if (has_loose) one(r.loose, r.part.loose(lane));
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int at = r.part.head + 4 * (lane + 32 * j);
            if (lane + 32 * j < n4 && pass(top_of(r.v[j]))) { one(r.v[j].x, at); one(r.v[j].y, at + 1); one(r.v[j].z, at + 2); one(r.v[j].w, at + 3); }
        }
    };
    auto in_front = [&](int v) {                                  // of the lanes in front of this one
        int sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += other;
        }
        return sum - v;
    };
    if (!fill) put([&](float v) { return v >= least; }, in_front(mine));
    else {
        const float above = unordered(bound + 1);                 // the next float: v >= above is v > least
        mine = reach(above);
        put([&](float v) { return v >= above; }, in_front(mine));
        n = (int)__reduce_add_sync(0xffffffffu, (unsigned)mine);
        // the first of those equal to it: in front of the quads, in them, behind them
        auto some = [&](bool a, bool b, bool c, bool d, int at) {
            const int m = a + b + c + d;
            int to = n + in_front(m);
            if (a) { if (to < k) list[to] = candidate(least, at); ++to; }
            if (b) { if (to < k) list[to] = candidate(least, at + 1); ++to; }
            if (c) { if (to < k) list[to] = candidate(least, at + 2); ++to; }
            if (d && to < k) list[to] = candidate(least, at + 3);
            n = min(k, n + (int)__reduce_add_sync(0xffffffffu, (unsigned)m));
        };
        some(lane < r.part.head && r.loose == least, false, false, false, lane);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const bool in = lane + 32 * j < n4;
            some(in && r.v[j].x == least, in && r.v[j].y == least, in && r.v[j].z == least, in && r.v[j].w == least, r.part.head + 4 * (lane + 32 * j));
        }
        some(lane >= r.part.head && has_loose && r.loose == least, false, false, false, r.part.loose(lane));
    }
    __syncwarp();
#pragma unroll 1
    for (int i = lane; i < n; i += 32) {
        const unsigned long long v = list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += list[j] > v;
        if (rank < k) f(rank, v);
    }
    __syncwarp();                                                 // before the next row's candidates come
}
// The warps of a row wait for one another.
template <int W>
__device__ __forceinline__ void row_sync() {
    if (W == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / (32 * W)), "n"(32 * W) : "memory");
}
// A row's list and the logits at its ids (where p has logits to look at), by the warp that has the row.
template <class P>
__device__ __forceinline__ void list_ready(TeacherList& l, const P& p, size_t row) {
    copies_wait<0>();
    __syncwarp();
    list_gather(l, p, row);
    copies_end();
    __syncwarp();
    list_terms(l, p);
    const bool twice = list_twice(l, p);
    if ((threadIdx.x & 31) == 0) l.twice = twice;
    copies_wait<0>();
    __syncwarp();
}
template <int W, int J, bool ENTROPY, RowWork WORK>
__global__ void __launch_bounds__(kRowThreads) short_rows_kernel(VocabRows p) {
    constexpr bool DISTILL = WORK == kList || WORK == kGrad, GRAD = WORK == kGrad, TOP = WORK == kTop;
    constexpr int G = kRowWarps / W;   // rows of a CTA at a time
    static_assert(!TOP || W == 1, "a warp seeks the largest of its row");
    grid_release();
    grid_wait();
    __shared__ TeacherList lists[DISTILL ? G : 1];
    __shared__ float3 sums[2][kRowWarps];
    __shared__ unsigned long long candidates[TOP ? kRowWarps : 1][kCandidates];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool lead = warp % W == 0;   // the warp that has the row's list and results
    TeacherList& list = lists[DISTILL ? warp / W : 0];
    const float up = GRAD ? load_behind(p.grad_out) * p.per_row : 0.0f;
    int turn = 0;
    for (size_t row = (size_t)blockIdx.x * G + warp / W; row < p.rows; row += (size_t)gridDim.x * G) {
        const float* x = p.logits + row * p.stride;
        if (DISTILL && lead) { list_fetch(list, p, row); copies_end(); }
        int token = -1;
        float x_token = 0.0f;
        if (!DISTILL && p.tokens != nullptr && lead && lane == 0) {
            token = load_behind(p.tokens + row);
            if (token < 0 || token >= p.cols) token = -1;
            else x_token = load_behind(x + token);
        }
        const ShortRow<W, J> r(x, p.cols);
        Stats<ENTROPY> st = r.template stats<ENTROPY>(p.c);
        if (DISTILL && lead) list_ready(list, p, row);            // before anything of this row may become its gradient (grad_logits == logits)
        if (W > 1) {
            if (lane == 0) sums[turn][warp] = make_float3(st.m, st.s, st.a);
            row_sync<W>();
            const float3 part = sums[turn][warp / W * W + (lane & (W - 1))];
            st.m = part.x; st.s = part.y; st.a = part.z;
            st.template join<W>(p.c);
            turn ^= 1;
        }
        const float m = st.m, s = st.s, log_s = logf(s);
        auto log_prob = [&](float value) { return s == 0.0f ? -INFINITY : (value - m) * p.inv_t - log_s; };      // s == 0: nothing is left of the row
        if (!DISTILL && lead && lane == 0) {
            if (p.row_stats != nullptr) { p.row_stats[2 * row] = m; p.row_stats[2 * row + 1] = s; }
            if (p.logprobs != nullptr) p.logprobs[row] = token < 0 ? 0.0f : log_prob(x_token);
            if (ENTROPY) p.entropy[row] = s == 0.0f ? 0.0f : log_s - st.a / s * kLn2;
        }
        if constexpr (TOP) {
            const size_t at = row * (size_t)p.n_top;
            auto put = [&](int rank, int id, float value) {
                if (p.top_ids != nullptr) p.top_ids[at + rank] = id;
                if (p.top_logprobs != nullptr) p.top_logprobs[at + rank] = value;
            };
            if (s == s) short_tops(r, p.n_top, candidates[warp], [&](int rank, unsigned long long c) { put(rank, (int)(0xffffffffu - (uint32_t)c), log_prob(unordered((uint32_t)(c >> 32)))); });
            else for (int i = lane; i < p.n_top; i += 32) put(i, -1, s);       // not a number
        }
        if (DISTILL && lead) list_result(p, list, row, m, s, list_loss(list, p.n_teacher, log_prob));
        if (GRAD) {
            const float sg = gradient_sum(s, list.sum);
            const bool none = sg == 0.0f || up == 0.0f;
            const ProbGrad value = {m, p.c, up / sg};
            r.write(p.grad_logits + row * p.stride, none, value);
            row_sync<W>();
            if (lead && !none) list_write(list, p.n_teacher, p.grad_logits + row * p.stride, 0, p.cols, up, value);
        }
        if (DISTILL) __syncwarp();                                // before the next row's list comes
    }
}
// The most probable tokens of a row that a CTA holds: one bound, of all the row, and what reaches it straight out of the registers.
template <int J, bool ENTROPY>
__global__ void __launch_bounds__(kRowThreads, 2) held_tops_kernel(VocabRows p) {
    grid_release();
    grid_wait();
    __shared__ Selection z;
    __shared__ float3 sums[2][kRowWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = p.n_top;
    if (threadIdx.x == 0) z.n_list[0] = z.n_list[1] = 0;
    int turn = 0;
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const float* x = p.logits + row * p.stride;
        int token = -1;
        float x_token = 0.0f;
        if (p.tokens != nullptr && threadIdx.x == kResultThread) {
            token = load_behind(p.tokens + row);
            if (token < 0 || token >= p.cols) token = -1;
            else x_token = load_behind(x + token);
        }
        const ShortRow<kRowWarps, J> r(x, p.cols);
        Stats<ENTROPY> st = r.template stats<ENTROPY>(p.c);
        if (lane == 0) sums[turn][warp] = make_float3(st.m, st.s, st.a);
        float top = r.loose;
#pragma unroll
        for (int j = 0; j < J; ++j) top = fmaxf(top, top_of(r.v[j]));
        const float least = unordered(max(bound_of(ordered(top), k, z.bound[turn]), ordered(-INFINITY)));      // a barrier in there: the sums are there too
        int* count = &z.n_list[turn];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = threadIdx.x + kRowThreads * j;
            if (i < r.part.n4 && top_of(r.v[j]) >= least) take(z, count, r.v[j], r.part.head + 4 * i, least, false);
        }
        if ((int)threadIdx.x < r.part.n - 4 * r.part.n4) take(z, count, alone(r.loose), r.part.loose(threadIdx.x), least, false);
        const float3 part = sums[turn][lane & (kRowWarps - 1)];
        st.m = part.x; st.s = part.y; st.a = part.z;
        st.template join<kRowWarps>(p.c);
        const float m = st.m, s = st.s, log_s = logf(s);
        auto log_prob = [&](float value) { return s == 0.0f ? -INFINITY : (value - m) * p.inv_t - log_s; };      // s == 0: nothing is left of the row
        if (threadIdx.x == kResultThread) {
            if (p.row_stats != nullptr) { p.row_stats[2 * row] = m; p.row_stats[2 * row + 1] = s; }
            if (p.logprobs != nullptr) p.logprobs[row] = token < 0 ? 0.0f : log_prob(x_token);
            if (ENTROPY) p.entropy[row] = s == 0.0f ? 0.0f : log_s - st.a / s * kLn2;
        }
        __syncthreads();
        int n = *count;
        if (threadIdx.x == 0) z.n_list[turn ^ 1] = 0;             // for the next row
        const size_t at = row * (size_t)k;
        auto put = [&](int rank, int id, float value) {
            if (p.top_ids != nullptr) p.top_ids[at + rank] = id;
            if (p.top_logprobs != nullptr) p.top_logprobs[at + rank] = value;
        };
        if (!(s == s)) {                                          // not a number: its places are not looked at
            if ((int)threadIdx.x < k) put(threadIdx.x, -1, s);
            continue;
        }
        if (n > kCandidates) n = take_few(z, count, r.part.p, r.part.n, 0, least, k, k);
        each_best(z.list, n, k, [&](int rank, unsigned long long c) { put(rank, (int)(0xffffffffu - (uint32_t)c), log_prob(unordered((uint32_t)(c >> 32)))); });
    }
}
template <int W, int J, bool DISTILL>
__global__ void __launch_bounds__(kRowThreads) short_grad_kernel(VocabGrad p) {
    constexpr int G = kRowWarps / W;
    grid_release();
    grid_wait();
    __shared__ TeacherList lists[DISTILL ? G : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool lead = warp % W == 0;
    TeacherList& list = lists[DISTILL ? warp / W : 0];
    for (size_t row = (size_t)blockIdx.x * G + warp / W; row < p.rows; row += (size_t)gridDim.x * G) {
        const float* x = p.logits + row * p.stride;
        float* g = p.grad_logits + row * p.stride;
        if (DISTILL && lead) { list_fetch(list, p, row); copies_end(); }
        const float m = load_behind(p.row_stats + 2 * row), s = load_behind(p.row_stats + 2 * row + 1);
        const Terms t = grad_terms<DISTILL>(p, row, m, s);
        const float x_token = lead && t.token >= 0 ? load_behind(x + t.token) : 0.0f;
        const ShortRow<W, J> r(x, p.cols);
        if (DISTILL && lead) list_ready(list, p, row);
        row_sync<W>();                                            // all that is read of the row, before any of it is written (grad_logits may be logits)
        const ProbGrad prob = {m, p.c, t.k0};
        const EntropyGrad with_entropy = {m, p.c, t.k0, t.k1};
        if (DISTILL) r.write(g, t.none, prob);
        else r.write(g, t.none, with_entropy);
        row_sync<W>();
        if (lead && !t.none) {
            if (DISTILL) list_write(list, p.n_teacher, g, 0, p.cols, t.up, prob);
            else if (lane == 0 && t.token >= 0) g[t.token] = with_entropy(x_token) + t.up;
        }
        if (DISTILL) __syncwarp();                                // before the next row's list comes
    }
}

// Attributes of a launch: overlapping with the one before it, and the CTAs of a row as a cluster.
template <class... P>
cudaError_t launch_rows(void (*kern)(P...), unsigned grid, int threads, int cluster, size_t smem, cudaStream_t stream, const P&... p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, p...);
}
// CTAs of a row: as many as leave none of the SMs idle, with 2048 logits each at least (one row of 32000: 6.8 us by eight, 16 rows 7.5).  Up to four on an SM (three
// with a selection's shared memory) where a CTA's part stays long enough to pay for the cluster's seam.  One / two CTAs: 200 x 128256 statistics 23 / 20 us, with 20 tops
// 33 / 26, lists' losses 27 / 22, but 150 x 50003 statistics 10.3 / 11.1 (from 61440 on, where one CTA
// takes a sixteenth step: 290 x 61400 14.8 / 16.9, 150 x 61400 11.1 / 11.8, 200 x 61500 14.5 / 13.3, 290 x 64000 16.1 / 15.0); the gradient, a second pass over what L2 holds of a row, gains from shorter
// parts on: 150 x 24000 19 / 17.6, 200 x 14000 14.4 / 12.8.
int row_cluster(const VocabRows& p, int sm_count) {
    const size_t most = p.n_top ? 3 : 4;
    const int least = p.grad_logits ? 6144 : p.n_top || p.n_teacher ? 24576 : 30720;
    int n = 1;
    while (n < kMaxCluster && ((p.rows * 2 * n <= 2 * (size_t)sm_count && p.cols / (2 * n) >= 2048) || (p.rows * 2 * n <= most * sm_count && p.cols / (2 * n) >= least))) n *= 2;
    return n;
}
// Up to how many columns.  11000 x 8192 by CTAs / by warps: statistics 60 / 77 us, lists' loss 80 / 82, the gradient of log probabilities 111 / 111, of lists 116 / 111, loss
// and gradient 225 / 128; 3000 x 16384 of these 77 in the ring / 75.  Fewer rows than three an SM: 300 x 2000 statistics 3.7 / 3.3 us, their gradient 3.3 / 3.9.
// With tokens sought: 600 x 2000 with 20 / 64 of them 9.1 / 9.0 us and 13 / 17 (four rows an SM), 11000 x 2000 99 / 46 and 143 / 81, 3000 x 1000 28 / 10 and 41 / 16.  Below 1024
// columns a CTA has warps without values, which leave it no bound: 1 x 500 18 / 5.5 us, 11000 x 500 769 / 19; 1 x 1024 4.5 / 6.3.  Statistics alone, which are
// the same bits then: 20 x 1000 2.6 / 2.6.
constexpr int kShortAll = 1023, kShortTop = 2048, kShortStats = 4096, kShortGrad = 4096, kShortListGrad = 8192, kShortBoth = 16384;
// f(warps of a row, quads of a lane) by the columns, MOST at most
template <int W, int J>
struct Short { static constexpr int warps = W, quads = J; };
template <int MOST, class F>
cudaError_t short_by_cols(int cols, F f) {
    if (cols <= 512) return f(Short<1, 4>());
    if (cols <= 1024) return f(Short<1, 8>());
    if constexpr (MOST > 4096) {
        if (cols > 8192) {
            if constexpr (MOST > 8192) return f(Short<8, 16>());
        }
        if (cols > 4096) return f(Short<4, 16>());
    }
    if constexpr (MOST > 2048) {
        if (cols > 2048) return f(Short<2, 16>());
    }
    return f(Short<1, 16>());
}
bool short_rows(size_t rows, int cols, int most, int sm_count) { return cols <= most && rows >= 3 * (size_t)sm_count; }
bool short_forward(const VocabRows& p, int sm_count) {
    if (p.n_teacher == 0 && p.cols <= kShortAll) return true;
    if (p.n_top) return short_rows(p.rows / 2, p.cols, kShortTop, sm_count);
    return short_rows(p.rows, p.cols, p.grad_logits ? kShortBoth : kShortStats, sm_count);
}
unsigned short_grid(size_t rows, int warps, int sm_count) {
    const size_t at_once = kRowWarps / warps, want = (rows + at_once - 1) / at_once, cap = (size_t)sm_count * 8;
    return (unsigned)(want < cap ? want : cap);
}
// Where rows are few, and no longer than a CTA holds: half the chain of a row (no bounds and notes on the way, no cluster).  Through vocab_rows_kernel / here, 20 tokens:
// 1 x 8000 6.5 / 4.5 us, 30 x 16384 7.8 / 6.5, 148 x 12345 10.1 / 6.5, 777 x 12345 21 / 19, 600 x 2000 9.1 / 9.6, 1184 x 12345 24.9 / 24.9, 4096 x 8000 56 / 59: a row takes
// registers that two or three CTAs an SM have, and no copies ahead.
bool held_tops(const VocabRows& p, int sm_count) {
    return p.n_top > 0 && p.cols > kShortAll && p.cols <= 64 * kRowThreads && p.rows <= (p.cols >= 4096 ? 6 : 3) * (size_t)sm_count;
}
cudaError_t launch_held_tops(const VocabRows& p, int sm_count, cudaStream_t stream) {
    const size_t cap = (size_t)sm_count * 4;
    const auto kern = p.cols <= 16 * kRowThreads ? (p.entropy ? held_tops_kernel<4, true> : held_tops_kernel<4, false>)
                    : p.cols <= 32 * kRowThreads ? (p.entropy ? held_tops_kernel<8, true> : held_tops_kernel<8, false>)
                                                 : (p.entropy ? held_tops_kernel<16, true> : held_tops_kernel<16, false>);
    return launch_rows(kern, (unsigned)(p.rows < cap ? p.rows : cap), kRowThreads, 1, 0, stream, p);
}
cudaError_t launch_forward(VocabRows& p, int sm_count, cudaStream_t stream) {
    if (held_tops(p, sm_count)) return launch_held_tops(p, sm_count, stream);
    if (short_forward(p, sm_count)) {
        const auto launch = [&](auto kern, int warps) { return launch_rows(kern, short_grid(p.rows, warps, sm_count), kRowThreads, 1, 0, stream, p); };
        if (p.grad_logits)
            return short_by_cols<kShortBoth>(p.cols, [&](auto w) { return launch(short_rows_kernel<decltype(w)::warps, decltype(w)::quads, false, kGrad>, w.warps); });
        if (p.n_top)
            return short_by_cols<kShortTop>(p.cols, [&](auto w) {
                return p.entropy ? launch(short_rows_kernel<1, decltype(w)::quads, true, kTop>, 1) : launch(short_rows_kernel<1, decltype(w)::quads, false, kTop>, 1);
            });
        return short_by_cols<kShortStats>(p.cols, [&](auto w) {
            constexpr int W = decltype(w)::warps, J = decltype(w)::quads;
            return p.n_teacher ? launch(short_rows_kernel<W, J, false, kList>, W) : p.entropy ? launch(short_rows_kernel<W, J, true, kPlain>, W) : launch(short_rows_kernel<W, J, false, kPlain>, W);
        });
    }
    p.cluster = row_cluster(p, sm_count);
    // Bounds after 1, 2, 4, 8, ... steps, between two of which there are as many hits again; after 1 and 2 only where a barrier and a bound are more than the
    // hits they save.  All of them / two, k = 20: 4096 x 32000 (8 steps) 112 / 110 us, 2000 x 50003 82 / 86, 600 x 128256 69 / 122; k = 64:
    // 147 / 139, 99 / 138, 76 / 140; k = 128, 4096 x 32000: 231 / 302, as two leave more than kHits.
    p.last_bound = p.n_top > 64 || p.cols / p.cluster > 10 * 4 * kQuads * kRowThreads ? INT_MAX - 1 : 1;
    const size_t cap = (size_t)sm_count * 4;
    const unsigned grid = p.cluster > 1 ? (unsigned)(p.rows * p.cluster) : (unsigned)(p.rows < cap ? p.rows : cap);
    const bool distill = p.n_teacher > 0;
    const size_t smem = kStreamBytes + (distill ? 3 * sizeof(TeacherList) : p.n_top ? sizeof(Selection) + (p.cluster > 1 ? kMaxCluster * kMaxList * sizeof(unsigned long long) : 0) : 0);
    const auto kern = distill ? (p.grad_logits ? vocab_rows_kernel<false, kGrad> : vocab_rows_kernel<false, kList>)
                    : p.n_top ? (p.entropy ? vocab_rows_kernel<true, kTop> : vocab_rows_kernel<false, kTop>)
                              : (p.entropy ? vocab_rows_kernel<true, kPlain> : vocab_rows_kernel<false, kPlain>);
    const cudaError_t e = smem <= 48 * 1024 - sizeof(RowShared) ? cudaSuccess : cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return e != cudaSuccess ? e : launch_rows(kern, grid, kRowThreads, p.cluster, smem, stream, p);
}
// Few chunks: each costs 1500 cycles of a row however small it is (4000 x 17800 in 2 / 4 / 8 of them 115 / 139 / 232 us).  But rows that come while one is at work need
// room: two chunks more than a row has beside the one that goes out, where up to seven leave it (4096 x 32000 in 4 / 5 / 6 / 8: 194 / 185 / 206 / 240 us;
// 4096 x 22000 in 2 / 3 / 4: 161 / 139 / 146), else as many as a row has (2500 x 40000 in 4 / 5 / 6: 158 / 157 / 169).  chunks = 0: too long.
Ring ring_of(int cols) {
    const int n4 = cols >> 2, all = (int)(kRingBytes / sizeof(float4));
    Ring r = {n4, 1, kRingAhead + 1};
    if (n4 * r.slots <= all) return r;
    for (int room = 2; room >= 0; room -= 2)
        for (r.chunks = 2; r.chunks <= (room ? 7 : kRingMost); ++r.chunks) {
            r.chunk = (n4 + r.chunks - 1) / r.chunks;
            r.slots = std::min((kRingAhead + 1) * r.chunks, all / r.chunk);
            if (r.slots - 1 >= r.chunks + room) return r;
        }
    return {0, 0, 0};
}
// Rows of at least 11264 logits (300 x 12000 with lists of 64: 16.2 us, twice out of L2 16.4; 3000 x 10000: 85 and 77; a row takes the list's warp 4 us however short
// it is) that are not for short_rows_kernel, as many as keep all SMs busy, gradients on the logits' 16-byte boundaries.
// Longer ones by as many CTAs as hold a row: more of them are more clusters' seams and fewer clusters that fit the GPU (1000 x 128256 by 3 / 4 / 6: 222 / 240 / 252 us,
// 400 x 262144 by 6 / 8: 193 / 223, 2000 x 60000 by 2 / 3: 190 / 223; twice out of L2 298, 256 and 285).
bool ring_takes(VocabRows& p, int sm_count, size_t max_smem) {
    const auto part = [&] { return ((p.cols + p.cluster - 1) / p.cluster + 3) & ~3; };
    for (p.cluster = 1; ring_of(part()).chunks == 0; ++p.cluster)
        if (p.cluster == kMaxCluster) return false;
    // few rows: in parts of no fewer than 11264 (200 x 32000 by one CTA 25 us, by two, twice out of L2, 21.6, by two here 18.2)
    while (p.rows * p.cluster < 2 * (size_t)sm_count && p.cluster < kMaxCluster && p.cols / (p.cluster + 1) >= 11264) ++p.cluster;
    return p.cols >= 11264 && !short_rows(p.rows, p.cols, kShortBoth, sm_count) && p.rows * p.cluster >= 2 * (size_t)sm_count && kRingBytes + kRingLists * sizeof(TeacherList) + 2048 <= max_smem &&
           ((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.grad_logits)) & 15) == 0;
}
cudaError_t launch_ring(VocabRows& p, int sm_count, cudaStream_t stream) {
    const auto kern = p.cluster > 1 ? distill_ring_kernel<true> : distill_ring_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes);
    if (e != cudaSuccess) return e;
    size_t at_once = sm_count;
    if (p.cluster > 1) {                              // as many as run at once: large ones do not fill every part of the GPU
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(p.cluster); cfg.blockDim = dim3(kRingThreads + 64); cfg.dynamicSmemBytes = kRingBytes;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = p.cluster; at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at; cfg.numAttrs = 1;
        int n = 0;
        if ((e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg)) != cudaSuccess) return e;
        at_once = n > 0 ? n : 1;
    }
    const Ring r = ring_of(((p.cols + p.cluster - 1) / p.cluster + 3) & ~3);
    return launch_rows(kern, (unsigned)((p.rows < at_once ? p.rows : at_once) * p.cluster), kRingThreads + 64, p.cluster, kRingBytes, stream, p, r);
}
void temperature_of(float t, float* c, float* inv_t) {
    *inv_t = 1.0f / t;
    *c = (float)(1.4426950408889634 / (double)t);
}
// One factor, so that no product on the way leaves fp32 where the result does not.
float per_row_of(float t, size_t rows) { return (float)(1.0 / ((double)t * (double)rows)); }
cudaError_t launch_grad(bool distill, VocabGrad& p, int sm_count, cudaStream_t stream) {
    if (short_rows(p.rows, p.cols, distill ? kShortListGrad : kShortGrad, sm_count)) {
        const auto launch = [&](auto kern, int warps) { return launch_rows(kern, short_grid(p.rows, warps, sm_count), kRowThreads, 1, 0, stream, p); };
        return distill ? short_by_cols<kShortListGrad>(p.cols, [&](auto w) { return launch(short_grad_kernel<decltype(w)::warps, decltype(w)::quads, true>, w.warps); })
                       : short_by_cols<kShortGrad>(p.cols, [&](auto w) { return launch(short_grad_kernel<decltype(w)::warps, decltype(w)::quads, false>, w.warps); });
    }
    // tiles of a row where the rows are fewer than the CTAs that fill the SMs
    const size_t want = 4 * (size_t)sm_count;
    p.tiles = 1;
    while (p.rows * (size_t)p.tiles < want && p.cols / (2 * p.tiles) >= 2048) p.tiles *= 2;
    p.per = ((p.cols + p.tiles - 1) / p.tiles + 3) & ~3;
    p.tiles = (p.cols + p.per - 1) / p.per;
    const size_t items = p.rows * (size_t)p.tiles, cap = (size_t)sm_count * 16;
    return launch_rows(distill ? vocab_grad_kernel<true> : vocab_grad_kernel<false>, (unsigned)(items < cap ? items : cap), kRowThreads, 1, 0, stream, p);
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
    return launch_forward(p, sm_count, stream);
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
                                     int n_teacher, float temperature, int* err_word, int sm_count, size_t max_smem, cudaStream_t stream) {
    VocabRows p = {};
    p.logits = logits; p.rows = rows; p.stride = stride; p.cols = cols;
    temperature_of(temperature, &p.c, &p.inv_t);
    p.teacher_ids = teacher_ids; p.teacher_logits = teacher_logits; p.n_teacher = n_teacher;
    p.losses = losses; p.row_stats = row_stats; p.grad_out = grad_out; p.per_row = per_row_of(temperature, rows); p.grad_logits = grad_logits;
    p.err_word = err_word;
    const cudaError_t e = grad_logits != nullptr && ring_takes(p, sm_count, max_smem) ? launch_ring(p, sm_count, stream) : launch_forward(p, sm_count, stream);
    return e != cudaSuccess ? e : launch_mean(losses, out, rows, rows, stream);
}
cudaError_t launch_distillation_loss_backward(const float* logits, const int* teacher_ids, const float* teacher_logits, const float* row_stats,
                                              const float* grad_out, float* grad_logits, size_t rows, int cols, size_t stride, int n_teacher,
                                              float temperature, int sm_count, cudaStream_t stream) {
    VocabGrad p = {};
    p.logits = logits; p.rows = rows; p.stride = stride; p.cols = cols;
    temperature_of(temperature, &p.c, &p.inv_t);
    p.teacher_ids = teacher_ids; p.teacher_logits = teacher_logits; p.n_teacher = n_teacher; p.row_stats = row_stats;
    p.grad_out = grad_out; p.inv_t = per_row_of(temperature, rows); p.grad_logits = grad_logits;
    return launch_grad(true, p, sm_count, stream);
}
}  // namespace mcl
