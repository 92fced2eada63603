// Log-probabilities of given tokens, with the entropy and the likeliest tokens of their rows, from logits.
//
// Formulas, for a row x of logits with maximum m, Z = sum_i exp(x_i - m):
//   logprob  = x[id] - m - log Z
//   entropy  = log Z - sum_i exp(x_i - m) (x_i - m) / Z
//   top      = the `top` largest x by (value, then lower id), each with x_i - m - log Z
// A logit of minus infinity has probability 0 and adds nothing.  A row with a NaN or plus infinity, or of minus infinities
// alone, has no distribution: its floats are NaN (with a NaN its ids are -1 and bit 0 of *status is raised).
//
// What bounds it: the logits' bytes, read once.  A block walks a row, or a cluster of 2, 4 or 8 blocks a row where rows are few
// (partial sums and candidates meet in the first block's shared memory), 16 logits a thread at a time, the next 16 on their way.
// Sums: a thread carries (m, Z, sum e (x - m)) of its own logits in 32 bits and rescales when a group of 16 raises m.
// Top: the first group's maxima, one for four threads, give a bound -- the `top`-th largest of them is at most the row's `top`-th largest
// -- and only logits at or above it, in the order of (value, lower id), go to a list in shared memory; after two groups, five and
// eleven the list's own `top`-th best is the bound.  At the end each of the list counts how many of it are in front.
// Logits are read once, but for two kinds of rows.  A minus infinity that no later rise of its thread's maximum drops makes w NaN, and w is made again over
// the block's part.  Where a list runs over (logits that rise along the row) the block finds the bound by bisection over its part.
// Measured: 2,046 rows of 50,257 float32 logits with the top 20 in 94 us, 4.4 TB/s or 67% of a copy's rate; with minus infinities 158; rising
// 7,900.  What bounds the 94 us is no one thing: 16 instructions a logit take half of the issue slots, memory is at half of its
// peak, and a warp waits (7 a scheduler) for its own last instruction, for memory, at barriers and for instructions in turn; 2,046 blocks are
// 1.7 rounds.  In bfloat16 91 us for half the bytes.  8 rows with the top 5 in 9.3 us: the launch, the first loads, three sorts
// of the bound and the cluster's join.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int EACH = 16;                   // logits a thread takes at a time
constexpr int LIST = 1024;                 // candidates a block keeps
constexpr int MAX_TOP = 32;
constexpr int GROUPS = 64;                 // of neighbouring threads, whose maxima give the first bound
constexpr int MAX_CLUSTER = 8;
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long u64;

// Value, then lower id, as one number that is larger for the one in front.  x + 0 makes one zero of two.
__device__ __forceinline__ u64 rank_key(float x, int id) {
    const unsigned b = __float_as_uint(x + 0.0f);
    const unsigned k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (u64)k << 32 | (unsigned)~id;
}
__device__ __forceinline__ float key_value(u64 key) {
    const unsigned k = (unsigned)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ int key_id(u64 key) { return (int)~(unsigned)key; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Sums {
    float m, z, w;      // maximum, sum of e^(x - m), sum of e^(x - m) (x - m)
};
// `s` with its maximum raised to m.  Where the factor is 0 the old sums are gone (and w + (..) z might be infinite).
__device__ __forceinline__ Sums raised(Sums s, float m) {
    if (m == s.m) return s;
    const float f = ex2((s.m - m) * LOG2E);
    if (f == 0.0f && s.z == s.z) return {m, 0.0f, 0.0f};
    return {m, s.z * f, (s.w + (s.m - m) * s.z) * f};
}
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    a = raised(a, m);
    b = raised(b, m);
    return {m, a.z + b.z, a.w + b.w};
}
__device__ __forceinline__ void add(Sums& s, float x) {       // x <= s.m, or not a number
    const float d = x - s.m, e = ex2(d * LOG2E);
    s.z += e;
    s.w = fmaf(e, fmaxf(d, -1e30f), s.w);                      // of minus infinity: e = 0, and 0 * d must be 0
}
// two 32-bit operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// What a block knows of its part of a row.
struct Part {
    Sums sums;
    int n_top;
    u64 top[MAX_TOP];
};

template <typename T, int THREADS>
struct Group {                                                  // a thread's 16 logits, as they come from memory
    static constexpr int PER = 16 / (int)sizeof(T), N = EACH / PER;
    uint4 raw[N];
    // pieces first, first + THREADS, .. of the row's 16-byte pieces; those at or past `end` are minus infinities
    __device__ __forceinline__ void load(const T* p, int first, int end) {
        if (first - (int)threadIdx.x + N * THREADS <= end) {     // all of them are there
            const uint4* from = reinterpret_cast<const uint4*>(p) + first;
#pragma unroll
            for (int u = 0; u < N; u++) raw[u] = __ldcs(from + u * THREADS);
            return;
        }
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int v = first + u * THREADS;
            const unsigned none = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
            raw[u] = v < end ? __ldcs(reinterpret_cast<const uint4*>(p) + v) : make_uint4(none, none, none, none);
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        const uint4 r = raw[i / PER];
        const int e = i % PER;
        if (sizeof(T) == 4) return __uint_as_float(e == 0 ? r.x : e == 1 ? r.y : e == 2 ? r.z : r.w);
        const unsigned w = e / 2 == 0 ? r.x : e / 2 == 1 ? r.y : e / 2 == 2 ? r.z : r.w;
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
};

// THREADS: 256, or 128 where every block has a row to itself: then twice as many rows are under way at a time, and what a row needs before
// and behind its walk is hidden behind the others'.  Rows of 50,257, 128 threads against 256: 2,046 rows 94 us and 110, 1,200 rows
// 63 and 60, 600 rows 36 and 38, 300 rows 28 and 23; 3,000 rows of 4,000: 29 and 41; 300 rows of 128,256: 58 and 42.  Up to 296 rows (148 SMs) a
// row is shared: 20 us for 296, 19 for 256.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logprobs_kernel(const T* __restrict__ logits, long long ld, int vocab, const int* __restrict__ ids, int top, float* __restrict__ logprob,
                float* __restrict__ entropy, int* __restrict__ top_ids, float* __restrict__ top_logprobs, int parts,
                int* __restrict__ status) {
    __shared__ u64 list[LIST];
    __shared__ u64 maxima[GROUPS];
    __shared__ u64 best[MAX_TOP];
    __shared__ Sums warp_sums[THREADS / 32];
    __shared__ Part got[MAX_CLUSTER];                           // in the first block of a cluster: every block's
    __shared__ u64 s_bound;
    __shared__ int s_count, s_nan;
    __shared__ unsigned s_counts[THREADS / 32];

    pdl_launch_dependents();
    pdl_wait();
    const int row_at = blockIdx.x / parts, part = blockIdx.x % parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* row = logits + (size_t)row_at * ld;
    // the row's 16-byte pieces, and in front of and behind them what is left; the first block takes that too
    constexpr int PER = Group<T, THREADS>::PER;
    const int head = min(vocab, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
    const T* body = row + head;
    const int pieces = (vocab - head) / PER, per_part = (pieces + parts - 1) / parts;
    const int begin = min(pieces, part * per_part), end = min(pieces, begin + per_part);
    const int tail = head + pieces * PER, loose = part == 0 ? head + vocab - tail : 0;      // at most 2 (PER - 1) < THREADS
    if (tid == 0) {
        s_count = 0;
        s_bound = 0;
        s_nan = 0;
    }
    const int given = ids ? ids[row_at] : -1;

    Group<T, THREADS> now, next;
    now.load(body, begin + tid, end);
    int my_loose = tid < loose ? (tid < head ? tid : tail + tid - head) : -1;
    const float loose_x = my_loose >= 0 ? to_f32(row[my_loose]) : -INFINITY;

    Sums s = {-3.402823466e38f, 0.0f, 0.0f};
    u64 bound = 0;
    float bound_x = -INFINITY;
    auto offer = [&](float x, int id) {
        const u64 key = rank_key(x, id);
        if (key < bound) return;
        const int at = atomicAdd(&s_count, 1);
        if (at < LIST) list[at] = key;
    };
    // The list's `top` best alone, in order; the last of them is the new bound.
    auto tighten = [&]() {
        __syncthreads();
        const int n = s_count;
        if (n > top && n <= LIST) {
            for (int i = tid; i < n; i += THREADS) {
                const u64 mine = list[i];
                int before = 0;
                for (int j = 0; j < n; j++) before += list[j] > mine;
                if (before < top) best[before] = mine;
            }
            __syncthreads();
            if (tid < top) list[tid] = best[tid];
            if (tid == 0) s_count = top;
            bound = best[top - 1];
            bound_x = key_value(bound);
        }
        __syncthreads();
    };
    float2 z = {0.0f, 0.0f}, w = {0.0f, 0.0f};                   // s.z and s.w, by the logits' parity
    int nth = 0;                                                  // groups of 16 taken
    int at = begin + tid;
    auto take = [&](const Group<T, THREADS>& now) {
        float part_most[4], most;                                // of its fours
#pragma unroll
        for (int q = 0; q < 4; q++) part_most[q] = fmaxf(fmaxf(now[4 * q], now[4 * q + 1]), fmaxf(now[4 * q + 2], now[4 * q + 3]));
        most = fmaxf(fmaxf(part_most[0], part_most[1]), fmaxf(part_most[2], part_most[3]));
        if (nth == 0 && top > 0) {
            // the `top`-th largest of the maxima of four threads each, loose logits among them
            u64 mine = my_loose >= 0 ? rank_key(loose_x, my_loose) : 0;
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const int v = at + i / PER * THREADS;
                if (v < end && now[i] == now[i]) mine = max(mine, rank_key(now[i], head + v * PER + i % PER));
            }
            constexpr int EACH_GROUP = THREADS / GROUPS;
#pragma unroll
            for (int o = 1; o < EACH_GROUP; o <<= 1) mine = max(mine, (u64)__shfl_xor_sync(0xffffffffu, mine, o));
            if (tid % EACH_GROUP == 0) maxima[tid / EACH_GROUP] = mine;
            __syncthreads();
            if (tid < GROUPS) {
                mine = maxima[tid];
                int before = 0;
#pragma unroll 16
                for (int j = 0; j < GROUPS; j++) before += maxima[j] > mine;
                if (before == top - 1 && mine) s_bound = mine;   // keys differ; with fewer than `top` the bound stays 0
            }
            __syncthreads();
            bound = s_bound;
            bound_x = bound ? key_value(bound) : -INFINITY;
            if (my_loose >= 0 && loose_x >= bound_x) offer(loose_x, my_loose);
        }
        nth++;
        // what the bound lets through falls with the logits it was taken from: after two groups, five and eleven it is taken anew
        if (top > 0 && (nth == 3 || nth == 6 || nth == 12)) tighten();
        if (most > s.m) {
            s.z = z.x + z.y;
            s.w = w.x + w.y;
            s = raised(s, most);
            z = {s.z, 0.0f};
            w = {s.w, 0.0f};
        }
        if (at - tid + Group<T, THREADS>::N * THREADS <= end) {
            const float2 minus = {-s.m, -s.m}, l2e = {LOG2E, LOG2E}, none = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < EACH; i += 2) {
                // of a logit of minus infinity e * d is 0 times infinity: the sum w becomes NaN and is made again behind the walk
                const float2 d = add2(make_float2(now[i], now[i + 1]), minus), t = fma2(d, l2e, none);
                const float2 e = {ex2(t.x), ex2(t.y)};
                z = add2(z, e);
                w = fma2(e, d, w);
            }
        } else {                                                  // the last ones, with minus infinities behind them
            Sums few = {s.m, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < EACH; i++) add(few, now[i]);
            z.x += few.z;
            w.x += few.w;
        }
        if (top > 0 && most >= bound_x) {
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (part_most[q] >= bound_x) {
#pragma unroll
                    for (int i = 4 * q; i < 4 * q + 4; i++) {
                        const int v = at + i / PER * THREADS;
                        if (now[i] >= bound_x && v < end) offer(now[i], head + v * PER + i % PER);
                    }
                }
        }
    };
    for (; nth == 0 || at - tid < end; at += THREADS * Group<T, THREADS>::N) {
        next.load(body, at + THREADS * Group<T, THREADS>::N, end);
        take(now);
        at += THREADS * Group<T, THREADS>::N;
        if (at - tid >= end) break;
        now.load(body, at + THREADS * Group<T, THREADS>::N, end);
        take(next);
    }
    s.z = z.x + z.y;
    s.w = w.x + w.y;
    if (my_loose >= 0) {
        if (loose_x > s.m) s = raised(s, loose_x);
        add(s, loose_x);
    }

    // ---- the block's sums ------------------------------------------------------------------------------------------
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums b = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o), __shfl_xor_sync(0xffffffffu, s.w, o)};
        s = joined(s, b);
    }
    if (lane == 0) warp_sums[warp] = s;
    __syncthreads();
    s = warp_sums[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; i++) s = joined(s, warp_sums[i]);

    if (s.w != s.w && s.z == s.z) {                              // minus infinities among the block's logits: w over its part again
        __syncthreads();
        Sums mine = {s.m, 0.0f, 0.0f};
        for (int v = begin + tid; v < end; v += THREADS)
            for (int e = 0; e < PER; e++) add(mine, to_f32(body[(size_t)v * PER + e]));
        if (my_loose >= 0) add(mine, loose_x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine.w += __shfl_xor_sync(0xffffffffu, mine.w, o);
        if (lane == 0) warp_sums[warp].w = mine.w;
        __syncthreads();
        s.w = 0.0f;
        for (int i = 0; i < THREADS / 32; i++) s.w += warp_sums[i].w;
    }

    // ---- the block's `top` best ----------------------------------------------------------------------------------------
    auto each = [&](auto&& f) {                                  // f(x, id) over the thread's share of the block's part, again
        for (int v = begin + tid; v < end; v += THREADS)
            for (int e = 0; e < PER; e++) f(to_f32(body[v * PER + e]), head + v * PER + e);
        if (my_loose >= 0) f(loose_x, my_loose);
    };
    if (s.z != s.z) {                                            // an infinity or a NaN: which of the two
        each([&](float x, int) { if (x != x) s_nan = 1; });
        __syncthreads();
    }
    const int n_here = (end - begin) * PER + loose, keep = min(top, n_here);
    if (top > 0 && s_count > LIST) {
        // the `keep`-th largest key, by bisection; there are at least `keep` keys above 0
        u64 lo = 0, hi = ~0ull;
        while (lo < hi) {
            const u64 mid = lo + ((hi - lo) >> 1) + 1;
            unsigned c = 0;
            each([&](float x, int id) { c += x == x && rank_key(x, id) >= mid; });
            c = __reduce_add_sync(0xffffffffu, c);
            __syncthreads();
            if (lane == 0) s_counts[warp] = c;
            __syncthreads();
            c = 0;
            for (int i = 0; i < THREADS / 32; i++) c += s_counts[i];
            if (c >= (unsigned)keep) lo = mid; else hi = mid - 1;
        }
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        bound = lo;
        each([&](float x, int id) { if (x == x) offer(x, id); });
        __syncthreads();
    }
    const bool alone = parts == 1;
    Part* to = &got[0];
    if (!alone) {
        cg::this_cluster().sync();                               // the first block is there
        to = cg::this_cluster().map_shared_rank(&got[0], 0) + part;
    }
    const int n_list = min(s_count, LIST);
    for (int i = tid; i < n_list; i += THREADS) {
        const u64 mine = list[i];
        int before = 0;
        for (int j = 0; j < n_list; j++) before += list[j] > mine;
        if (before < keep) to->top[before] = mine;
    }
    if (tid == 0) {
        to->sums = s;
        to->n_top = s_nan ? -1 : min(keep, n_list);
    }
    if (alone) {
        __syncthreads();
    } else {
        cg::this_cluster().sync();
        if (part != 0) return;
    }

    // ---- the row's results -------------------------------------------------------------------------------------------
    Sums all = got[0].sums;
    bool has_nan = got[0].n_top < 0;
    for (int i = 1; i < parts; i++) {
        all = joined(all, got[i].sums);
        has_nan |= got[i].n_top < 0;
    }
    const float log_z = logf(all.z);
    if (tid == 0) {
        const bool there = given >= 0 && given < vocab;
        if (logprob) logprob[row_at] = there ? to_f32(row[given]) - all.m - log_z : given == -1 ? 0.0f : __uint_as_float(0x7fffffffu);
        if (entropy) entropy[row_at] = log_z - all.w / all.z;
        if (status && (has_nan || (!there && given != -1))) atomicOr(status, 1);
    }
    for (int i = tid; i < parts * MAX_TOP; i += THREADS) {
        const int p = i / MAX_TOP, k = i % MAX_TOP;
        if (k >= got[p].n_top && !has_nan) continue;
        if (has_nan) {
            if (p == 0 && k < top) {
                top_ids[(size_t)row_at * top + k] = -1;
                top_logprobs[(size_t)row_at * top + k] = __uint_as_float(0x7fffffffu);
            }
            continue;
        }
        const u64 mine = got[p].top[k];
        int before = k;                                          // a part's are in order
        for (int r = 0; r < parts; r++)
            if (r != p)
                for (int j = 0; j < got[r].n_top; j++) before += got[r].top[j] > mine;
        if (before < top) {
            top_ids[(size_t)row_at * top + before] = key_id(mine);
            top_logprobs[(size_t)row_at * top + before] = key_value(mine) - all.m - log_z;
        }
    }
}

}  // namespace

// logits: [n_rows, vocab] of dtype, row pitch ld (elements).  ids: int32 [n_rows], -1 for a row without a given token (its logprob
// is 0); null: none.  logprob, entropy: float32 [n_rows], may be null.  top_ids (int32), top_logprobs (float32): [n_rows, top], top
// at most 32 and at most vocab.  Bit 0 of *status (may be null): an id outside the vocabulary (its logprob is NaN) or a NaN.
SANDY_API int sandy_token_logprobs(const void* logits, long long ld, int n_rows, int vocab, const int* ids, int top, float* logprob,
                                   float* entropy, int* top_ids, float* top_logprobs, int dtype, int* status, cudaStream_t stream) {
    if (n_rows == 0) return SANDY_OK;
    if (!logits || n_rows < 0 || vocab < 1 || top < 0 || (top > 0 && (!top_ids || !top_logprobs)) || (logprob && !ids)) return SANDY_ERR_ARGUMENT;
    if (top > MAX_TOP || top > vocab || (dtype != SANDY_F32 && dtype != SANDY_BF16)) return SANDY_ERR_UNSUPPORTED;
    // a row's pieces start on 16 bytes wherever its first logit lies, as long as that is a whole number of logits
    if ((uintptr_t)logits % (dtype == SANDY_F32 ? 4 : 2)) return SANDY_ERR_UNSUPPORTED;
    // Few rows: blocks share one, each with at least a group of 4,096 logits.
    int parts = 1;
    while (parts < MAX_CLUSTER && (long long)n_rows * parts * 2 <= 4ll * sandy_sm_count() && vocab / (parts * 2) >= 256 * EACH) parts *= 2;
    if ((long long)n_rows * parts > 0x7fffffffll) return SANDY_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_rows * parts));
    const int threads = parts > 1 ? 256 : 128;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (parts > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = parts;
        attr[na].val.clusterDim.y = 1;
        attr[na].val.clusterDim.z = 1;
        na++;
    }
    if (sandy_pdl_enabled()) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    cudaError_t e;
#define LAUNCH(T, THREADS)                                                                                                       \
    e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T, THREADS>, (const T*)logits, ld, vocab, ids, top, logprob, entropy, top_ids,  \
                           top_logprobs, parts, status)
    if (dtype == SANDY_F32) {
        if (threads == 256) LAUNCH(float, 256);
        else LAUNCH(float, 128);
    } else {
        if (threads == 256) LAUNCH(bf16, 256);
        else LAUNCH(bf16, 128);
    }
#undef LAUNCH
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
