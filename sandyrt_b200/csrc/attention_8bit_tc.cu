// Causal attention of prompt portions over the paged cache in 8 bits (kv_8bit.cuh) on the tcgen05 tensor cores: bfloat16 queries,
// heads of up to 128 (in the place of 64 or 128), pages of a multiple of 16 keys.
//
// Formula and scales as in attention_8bit.cu; the products are half-precision ones here too: codes are half-precision numbers without
// rounding, a query row is scaled by a power of two so that its largest element lies in [1, 2), and the scales of keys and values, which
// are the same for 16 keys of a tile at least, never touch an operand:
//   x_j = S_j * (sk * 2^eq * scale * log2 e) + log2 sv        p_j sv = 2^(x_j - M)       l += (sum over the run of 2^(x_j - M)) / sv
// With the maximum of a run taken over S, a score costs what it costs without scales: a maximum, an fma, an exponential, an addition.
//
// A block owns 256 query rows -- the heads of a group for consecutive tokens, row = token * group + head -- of one request's key/value
// head, as two tiles of 128 (tensor-memory lanes), and walks the keys in tiles of 128 which both share:
//   warps 0-3, 4-7   softmax of the two tiles, a thread a row: it reads its 128 scores with tcgen05.ld, and writes its weights as
//                    half-precision pairs over the first half of them with tcgen05.st;
//   warps 8-11       bring the codes (16 bytes a thread at a time, the next tile's while this one's are being written), turn
//                    them into half-precision numbers, and write them into shared memory as the operands lie there: K rows of 128
//                    bytes in the 128-byte swizzle, V likewise (an MN-major operand); rows past the portion's last key are zeros;
//   warp 12          issues the products: S of one tile while the other's softmax runs.  P lies where S lay, so that S of the next
//                    key tile follows P V of this one; both tiles' S and O fill the 512 columns of tensor memory at heads of 128.
// Head sizes between are the next of 64 and 128 with zeros behind their dims, in shared memory alone: 12 requests of 800 tokens behind
// 1,000, 9 heads of 48, 105 us (the mma.sync kernel 492); 12 prompts of 400, 12 heads of 80, 33 (173); 8 heads of 16, 500 tokens, 13 (24).
// The accumulators stay in tensor memory over all tiles and are rescaled there only when a row's maximum is more than 2^14 above its
// reference, which then goes to 2^-7 of the maximum (attention_8bit.cu; P stays below 2^14).  When S of a tile is there, the products before it are complete: O is at rest then.
//
// What bounds it: 32,768 exponentials a pair of tiles are 2,048 cycles of the special-function units, the products at heads of 128
// as much of the tensor cores; converting 32,768 codes is some 700 (int8) issue slots of each SM quarter.  256 rows a block halve the
// conversion's share and the reads of the cache.  One block an SM (193 KB of shared memory at heads of 128).
// Measured: 2,048 tokens behind 6,000, 32 heads of 128 reading 8 (int8): 288 us, 49% of the 1.67 PFLOP/s that a matrix product gets;
// four prompts of 500 to 950 tokens, 12 heads of 64 (e4m3): 32.6 us.  At heads of 64 a pair of tiles takes 3,300 cycles: 2,200 of softmax,
// and 1,100 from the weights to the next scores (the issuing warp's wake-up, two products, the way back), of which the two tiles
// overlap about half.  A block needs 6,500 cycles to its first scores (page, scale, codes, each a trip to memory) and 2,000 for its
// write-back; 256 blocks on 148 SMs are two rounds.  Blocks with the most keys start first, over all requests.
//
// Where blocks are fewer than SMs, clusters of 2, 4 or 8 share the key tiles of a block of rows.  Each block leaves its O (in the place of
// its keys and values) and its rows' M and l in its shared memory; then each joins its share of the rows, in the blocks' order.
//
// Every wait on an mbarrier is bounded; one that runs out raises bit 8 of the status word and the block ends without waiting again.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "cache8.h"
#include "kv_8bit.cuh"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int BN = 128;                  // keys of a tile
constexpr int THREADS = 416;
constexpr int FIRST_PRODUCER = 256, ISSUE_WARP = 12;
constexpr int STAGES = 2;
constexpr int CONSTS = 8;                // key tiles whose scales and pages are kept
constexpr float RESCALE = 14.0f, HEADROOM = 7.0f;     // of a row's reference, see attention_8bit.cu
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t HALF_TILE = 128 * 128;            // 128 rows of 64 half-precision numbers

constexpr uint32_t idesc_f16(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24); }

struct Args {
    const bf16* q;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const int *block_table, *q_start, *kv_before;
    bf16* out;
    int* status;
    const float *sink, *out_gate;
    const bf16* elem_gate;
    long long ld_q, ld_out, page_stride, scale_stride;
    int max_blocks, n_rows, max_n, n_heads, n_kv_heads, group, page_size, page_shift, num_pages;
    int window, keep_first, chunk, ld_elem_gate, gate_dim, splits, head_dim;
    float scale, softcap;
};

// What a run of 16 keys gives to its scores: the key's scale, log2 of the value's, one over it.
struct __align__(16) RunConsts {
    float ks, ev, inv, unused;
};

__device__ __forceinline__ void umma_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}" ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// One arrival for a warp whose lanes have all fenced what they wrote.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
// two 32-bit operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// HD: 64 or 128, the head size, or (FULL false) the next of the two above it: what is behind the head's dims is zeros in shared memory.
// SPLIT: a cluster of a.splits blocks shares a block's rows, each with a run of their key tiles.
template <int CODE, int HD, bool FULL, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) prefill_8bit_kernel(const __grid_constant__ Args a) {
    const int D = FULL ? HD : a.head_dim;
    constexpr int SUBS = HD / 64;                        // runs of 64 dims: 128-byte rows
    constexpr uint32_t Q_BYTES = SUBS * HALF_TILE, KV_BYTES = SUBS * HALF_TILE;
    constexpr uint32_t OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + STAGES * KV_BYTES;
    auto s_col = [](int g) { return (uint32_t)(128 * g); };           // columns of tensor memory: scores, later weights; results
    auto o_col = [](int g) { return (uint32_t)(256 + HD * g); };
    constexpr uint32_t IDESC_S = idesc_f16(BN), IDESC_PV = idesc_f16(HD) | (1u << 16);        // V: MN-major
    extern __shared__ uint8_t smem_raw[];
    __shared__ RunConsts s_consts[CONSTS][BN / 16];
    __shared__ long long s_off[CONSTS][BN / 16];         // where a run's rows lie in keys and values (page 0's, if nowhere)
    __shared__ unsigned s_runs[CONSTS];                  // the tile's runs: bit i, it has a page; bit 8 + i, its values' scale is not 2^ev
    __shared__ float s_rest[CONSTS][BN / 16];            // of these: the scale over 2^ev
    __shared__ uint64_t q_ready[2], first_k, k_empty[STAGES], v_empty[STAGES], s_full[2], go[2][2], o_full[2], c_full[CONSTS];
    __shared__ float2 s_ml[SPLIT ? 256 : 1];             // M and l of the rows
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_failed;

    pdl_launch_dependents();
    pdl_wait();
    // tiles in the slowest dimension: all requests' blocks with the most keys start first, and what is left for the end is small
    const int z = blockIdx.y, kvh = SPLIT ? blockIdx.x / a.splits : blockIdx.x, nth = blockIdx.z;
    const int rank = SPLIT ? blockIdx.x - kvh * a.splits : 0;
    const int row0 = a.q_start[z], n = a.q_start[z + 1] - row0, before = a.kv_before[z];
    // the portion's rows, blocks for them, and positions that are ints
    const bool there = row0 >= 0 && n <= a.n_rows - row0 && n <= a.max_n && (long long)before + n - 1 <= 0x7fffffffll;
    if (!there && n > 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, 16);
    const int tiles = there && n > 0 ? (int)(((long long)n * a.group + 255) / 256) : 0;
    if (nth >= tiles) return;
    const int first = (tiles - 1 - nth) * 256;
    const int n_valid = min(256, n * a.group - first);
    const int groups = n_valid > 128 ? 2 : 1;
    const int pos_first = before + first / a.group, pos_last = before + (first + n_valid - 1) / a.group;
    auto first_key = [&](int pos) {
        int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
        if (a.chunk > 0) lo = max(lo, pos - pos % a.chunk);
        return lo;
    };
    const int lo_first = first_key(max(pos_first, 0)), lo_last = first_key(max(pos_last, 0));
    // positions behind the block table's end have no page: no tile is walked for them, however far they are
    const long long in_table = (long long)a.max_blocks * a.page_size;
    const int key_last = (int)min((long long)pos_last, in_table - 1);
    if (key_last < pos_last && threadIdx.x == 0 && a.status) atomicOr(a.status, 16);
    const int kt_window = lo_first / BN;
    const int kept_tiles = lo_first > 0 ? min((int)((min((long long)a.keep_first, in_table) + BN - 1) / BN), kt_window) : 0;
    const int n_all = pos_last >= 0 ? kept_tiles + max(key_last / BN - kt_window + 1, 0) : 0;
    const int share = SPLIT ? (n_all + a.splits - 1) / a.splits : n_all, begin = SPLIT ? min(n_all, rank * share) : 0;
    const int n_it = SPLIT ? min(share, n_all - begin) : n_all;
    auto first_of = [&](int it) {
        const int t = begin + it;
        return (t < kept_tiles ? t : t - kept_tiles + kt_window) * BN;
    };
    const int tid = threadIdx.x, warp = tid >> 5;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;

    if (tid == 0) {
        for (int g = 0; g < 2; g++) {
            mbar_init(&q_ready[g], 4);
            mbar_init(&s_full[g], 1);
            // per tile of rows and parity of the key tile: its weights, V of the key tile and K of the next are there
            mbar_init(&go[g][0], 12);
            mbar_init(&go[g][1], 12);
            mbar_init(&o_full[g], 1);
        }
        mbar_init(&first_k, 4);
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < CONSTS; i++) mbar_init(&c_full[i], BN / 16);
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == ISSUE_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    auto wait_for = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity) || s_failed) return;
        if (!mbar_wait(bar, parity)) {
            if (a.status) atomicOr(a.status, 256);
            s_failed = 1;
        }
    };

    if (warp < 8) {
        // ---- softmax ------------------------------------------------------------------------------------------------
        const int g = warp >> 2, r = tid & 127;          // which tile; which row of it, the tensor-memory lane
        const int at = first + g * 128 + r;              // of the (request, key/value head)'s rows
        const bool mine = g * 128 + r < n_valid;
        const int token = mine ? at / a.group : 0, h = kvh * a.group + (mine ? at - token * a.group : 0);
        const int pos = mine ? before + token : -1;
        const int lo = first_key(max(pos, 0));
        float factor = 0.0f;
        if (g < groups) {
            // the row of q, scaled, as the first operand: 16-byte piece c of its 128-byte rows at piece c ^ (r & 7)
            const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(row0 + token) * a.ld_q + (size_t)h * D);
            uint4 w[HD / 8];
#pragma unroll
            for (int c = 0; c < HD / 8; c++) w[c] = mine && (FULL || 8 * c < D) ? src[c] : make_uint4(0u, 0u, 0u, 0u);
            uint32_t amax = 0;
#pragma unroll
            for (int c = 0; c < HD / 8; c++) {
                const uint32_t m = __vmaxu2(__vmaxu2(w[c].x & 0x7fff7fffu, w[c].y & 0x7fff7fffu), __vmaxu2(w[c].z & 0x7fff7fffu, w[c].w & 0x7fff7fffu));
                amax = max(amax, max(m & 0xffffu, m >> 16));
            }
            const int e2 = max(-100, min(120, (int)(amax >> 7) - 127));
            const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
            factor = __uint_as_float((uint32_t)(127 + e2) << 23) * a.scale * (a.softcap > 0.0f ? 1.0f : LOG2E);
            const uint32_t to = base + g * Q_BYTES + r * 128;
#pragma unroll
            for (int c = 0; c < HD / 8; c++) {
                auto two = [&](uint32_t x) { return pack_half(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xffff0000u) * down); };
                sts128(to + (c >> 3) * HALF_TILE + (((c & 7) ^ (r & 7)) << 4), two(w[c].x), two(w[c].y), two(w[c].z), two(w[c].w));
            }
            fence_async_proxy();
            warp_arrive(&q_ready[g]);
        }
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        float M = -INFINITY, l = 0.0f;
        // of the warp's rows: the first and the last position, the first visible key behind the kept ones
        const int pos_min = __reduce_min_sync(0xffffffffu, mine ? pos : 0x7fffffff), pos_max = __reduce_max_sync(0xffffffffu, pos);
        const int lo_min = __reduce_min_sync(0xffffffffu, mine ? lo : 0x7fffffff), lo_max = __reduce_max_sync(0xffffffffu, mine ? lo : 0);
        for (int it = 0; it < n_it && g < groups; it++) {
            const int j0 = first_of(it);
            wait_for(&c_full[it % CONSTS], (it / CONSTS) & 1);       // long there
            wait_for(&s_full[g], it & 1);
            tc_fence_after();
            uint32_t s[64];                              // half of the tile's scores at a time; later its weights, as pairs
            const RunConsts* consts = s_consts[it % CONSTS];
            auto read = [&](int half) {
                tmem_ld_32x32(lanes + s_col(g) + 64 * half, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
                tmem_ld_32x32(lanes + s_col(g) + 64 * half + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
                tmem_wait_ld();
            };
            // A tile that every row of the block sees whole needs no mask.  In any other the scores become x where they lie, 32 keys at a
            // time: not those that none of the warp's rows sees, and with a test a key only where some see it and some don't.
            const bool whole = j0 + BN - 1 <= pos_first && j0 >= lo_last && a.softcap == 0.0f;
            unsigned hidden = 0;                         // which 32 keys no row of the warp sees
            float top = -INFINITY;
            if (whole) {
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
                    read(half);
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        float m0 = __uint_as_float(s[16 * u]), m1 = __uint_as_float(s[16 * u + 1]);
#pragma unroll
                        for (int e = 2; e < 16; e += 2) {
                            m0 = fmaxf(m0, __uint_as_float(s[16 * u + e]));
                            m1 = fmaxf(m1, __uint_as_float(s[16 * u + e + 1]));
                        }
                        top = fmaxf(top, fmaf(fmaxf(m0, m1), consts[4 * half + u].ks * factor, consts[4 * half + u].ev));
                    }
                }
            } else {
#pragma unroll 1
                for (int q = 0; q < 4; q++) {
                    const int j = j0 + 32 * q;
                    if (j > pos_max || (j + 31 < lo_min && j >= a.keep_first)) {
                        hidden |= 1u << q;
                        continue;
                    }
                    uint32_t x[32];
                    tmem_ld_32x32(lanes + s_col(g) + 32 * q, x);
                    tmem_wait_ld();
                    const RunConsts c0 = consts[2 * q], c1 = consts[2 * q + 1];
                    float f0 = c0.ks * factor, f1 = c1.ks * factor;
                    if (a.softcap > 0.0f) {
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            x[e] = __float_as_uint(a.softcap * LOG2E * tanh_fast(__fdividef(__uint_as_float(x[e]) * (e < 16 ? f0 : f1), a.softcap)));
                        f0 = f1 = 1.0f;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e++) x[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), e < 16 ? f0 : f1, e < 16 ? c0.ev : c1.ev));
                    if (j + 31 > pos_min || j < lo_max) {
                        const int last = pos - j, from = lo - j, kept = a.keep_first - j;      // this row sees e <= last, e >= from or e < kept
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (e > last || (e < from && e >= kept)) x[e] = 0xff800000u;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e++) top = fmaxf(top, __uint_as_float(x[e]));
                    tmem_st_32x32(lanes + s_col(g) + 32 * q, x);
                }
                tmem_wait_st();
            }
            const bool move = top > M + RESCALE;
            if (__any_sync(0xffffffffu, move)) {
                const float next = top - HEADROOM, alpha = move ? ex2(M - next) : 1.0f;      // 0 on the row's first keys
                if (it > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD / 16; c++) {
                        uint32_t o[16];
                        tmem_ld_32x16(lanes + o_col(g) + 16 * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st_32x16(lanes + o_col(g) + 16 * c, o);
                    }
                    tmem_wait_st();
                }
                l *= alpha;
                if (move) M = next;
            }
            const float m_use = M == -INFINITY ? 0.0f : M;           // no key yet: weights are 2^-inf
            if (whole) {
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
                    read(half);
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const RunConsts c = consts[4 * half + u];
                        const float f = c.ks * factor, off = c.ev - m_use;
                        float2 sum = {0.0f, 0.0f};
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            float2 x = fma2(make_float2(__uint_as_float(s[16 * u + e]), __uint_as_float(s[16 * u + e + 1])), make_float2(f, f), make_float2(off, off));
                            x.x = ex2(x.x);
                            x.y = ex2(x.y);
                            sum = add2(sum, x);
                            s[8 * u + e / 2] = pack_half(x.x, x.y);
                        }
                        l = fmaf(sum.x + sum.y, c.inv, l);
                    }
                    // over columns whose scores have been read: 0..31 of the tile's 128, then 32..63
                    tmem_st_32x32(lanes + s_col(g) + 32 * half, s);
                }
            } else {
                // 32 keys' weights over 16 columns, whose scores have been read
#pragma unroll 1
                for (int q = 0; q < 4; q++) {
                    uint32_t x[32];
                    if ((hidden >> q) & 1) {
#pragma unroll
                        for (int e = 0; e < 16; e++) x[e] = 0u;
                    } else {
                        tmem_ld_32x32(lanes + s_col(g) + 32 * q, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            float2 sum = {0.0f, 0.0f};
#pragma unroll
                            for (int e = 16 * u; e < 16 * u + 16; e += 2) {
                                const float2 w = {ex2(__uint_as_float(x[e]) - m_use), ex2(__uint_as_float(x[e + 1]) - m_use)};
                                sum = add2(sum, w);
                                x[e / 2] = pack_half(w.x, w.y);
                            }
                            l = fmaf(sum.x + sum.y, consts[2 * q + u].inv, l);
                        }
                    }
                    tmem_st_32x16(lanes + s_col(g) + 16 * q, x);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&go[g][it & 1]);
        }
        if (SPLIT && g < groups) {
            // this block's sums where its keys and values lay, 4 dims of a row in a piece, a row's pieces 256 pieces apart
            if (n_it > 0) {
                wait_for(&o_full[0], 0);                             // of both: nothing reads keys and values any more
                if (groups == 2) wait_for(&o_full[1], 0);
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t o[32];
                    tmem_ld_32x32(lanes + o_col(g) + 32 * c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        sts128(base + OFF_K + ((8 * c + e) * 256 + tid) * 16, o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
            }
            s_ml[tid] = make_float2(M, l);
        }
        if (!SPLIT && g < groups) {
            if (n_it > 0) {
                wait_for(&o_full[g], 0);
                tc_fence_after();
            }
            const bool nothing = M == -INFINITY && l == 0.0f;        // no visible key
            if (a.sink && M > -INFINITY) l += ex2(fmaf(a.sink[h], LOG2E, -M));
            float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;        // no visible key: zeros
            if (a.out_gate && mine) inv *= a.out_gate[(size_t)(row0 + token) * a.n_heads + h];
            bf16* dst = a.out + (size_t)(row0 + token) * a.ld_out + (size_t)h * D;
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
                uint32_t o[32];
                if (n_it > 0) {
                    tmem_ld_32x32(lanes + o_col(g) + 32 * c, o);
                    tmem_wait_ld();
                }
                if (mine) {
                    float y[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) y[e] = nothing ? 0.0f : __uint_as_float(o[e]) * inv;
                    // one branch around all of it: a test at each element, and the code it jumps over, made the write-back three times as long
                    if (a.elem_gate) {
#pragma unroll
                        for (int e = 0; e < 32; e++) y[e] *= elem_gate_of(a.elem_gate, a.ld_elem_gate, a.gate_dim, row0 + token, h, 32 * c + e);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        if (FULL || 32 * c + e < D) *reinterpret_cast<uint4*>(dst + 32 * c + e) = make_uint4(pack_bf16(y[e], y[e + 1]), pack_bf16(y[e + 2], y[e + 3]),
                                                                                 pack_bf16(y[e + 4], y[e + 5]), pack_bf16(y[e + 6], y[e + 7]));
                }
            }
        }
    } else if (warp < ISSUE_WARP) {
        // ---- codes into operands ----------------------------------------------------------------------------------------
        constexpr int PIECES = HD / 16, STEP = 128 / PIECES, EACH = 128 / STEP;      // 16-byte pieces of a row; rows at a time; a thread's
        const int p = tid - FIRST_PRODUCER, piece = p % PIECES, my_row = p / PIECES;
        const int* table = a.block_table + (size_t)z * a.max_blocks;
        auto seen = [&](int j) { return j <= pos_last && (j >= lo_first || j < a.keep_first); };
        // Pages and scales of four tiles' runs, a lane of the first warp each: the pages are asked for four tiles ahead, the scales a
        // tile later, and noted another tile later, so that no one waits for the chain from the table to the scales.  A run whose values'
        // scale is not finite takes a key scale of NaN: rows that see it become NaN.
        int run_page = -1;
        float run_ks = 0.0f, run_vs = 0.0f;
        auto run_key = [&](int it) { return first_of(it + (p >> 3)) + 16 * (p & 7); };
        auto run_seen = [&](int it) {
            const int j = run_key(it);
            return it + (p >> 3) < n_it && j <= pos_last && (j + 15 >= lo_first || j < a.keep_first);
        };
        auto block_of = [&](int j) { return a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size; };
        auto ask_pages = [&](int it) {
            run_page = -1;
            if (run_seen(it)) {
                const int b = block_of(run_key(it));
                if (b < a.max_blocks) run_page = table[b];
                if (run_page >= a.num_pages) run_page = -1;
            }
        };
        auto ask_scales = [&]() {
            if (run_page < 0) return;
            run_vs = a.v_scale[(size_t)run_page * a.scale_stride + kvh];
            run_ks = a.k_scale[(size_t)run_page * a.scale_stride + kvh];
        };
        // The tiles' slots are free: two tiles before the first of them the products have left the tile eight before the last.
        auto note = [&](int it) {
            RunConsts c = {0.0f, -INFINITY, 0.0f, 0.0f};             // keys of no page weigh nothing
            long long off = 0;
            float rest = 1.0f;
            bool odd = false;
            const int slot = (it + (p >> 3)) % CONSTS;
            if (run_page >= 0) {
                const int j = run_key(it), biased = (int)(__float_as_uint(run_vs) >> 23) & 255, e = biased == 255 ? 127 : max(biased, 127 - 60);
                off = run_page * a.page_stride + ((long long)kvh * a.page_size + (j - block_of(j) * a.page_size)) * D;
                c.ks = biased == 255 ? __uint_as_float(0x7fffffffu) : run_ks;
                c.ev = (float)(e - 127);                             // at least -60: see attention_8bit.cu
                c.inv = __uint_as_float((unsigned)max(254 - e, 0) << 23);
                odd = biased != 255 && __float_as_uint(run_vs) != (unsigned)e << 23;
                rest = run_vs * c.inv;
            } else if (run_seen(it) && a.status) {
                atomicOr(a.status, 16);
            }
            const unsigned good = __ballot_sync(0xffffffffu, run_page >= 0), odds = __ballot_sync(0xffffffffu, odd);
            if (it + (p >> 3) < n_it) {
                s_consts[slot][p & 7] = c;
                s_off[slot][p & 7] = off;
                s_rest[slot][p & 7] = rest;
                if ((p & 7) == 0) s_runs[slot] = ((good >> p) & 0xff) | ((odds >> p) & 0xff) << 8;
                mbar_arrive(&c_full[slot]);
            }
        };
        // A thread's pieces of a tile; bit i of the result: piece i is one that counts.  The others are read from where something is, so
        // that no load hangs on a condition, and become zeros when stored.
        auto load = [&](const uint8_t* from, int it, uint4 (&w)[EACH]) {
            if (it >= n_it) return 0u;
            const int j0 = first_of(it), at = it % CONSTS;
            const unsigned good = s_runs[at] & 0xff;
            unsigned counts = (1u << EACH) - 1;
            if (good != 0xff || j0 + BN - 1 > pos_last || j0 < lo_first) {       // not every key has a page and is seen by a query
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    const int row = i * STEP + my_row;
                    if (!((good >> (row >> 4)) & 1) || !seen(j0 + row)) counts &= ~(1u << i);
                }
            }
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const int row = i * STEP + my_row;
                w[i] = __ldg(reinterpret_cast<const uint4*>(from + s_off[at][row >> 4] + ((row & 15) * D + (FULL || piece * 16 < D ? piece * 16 : 0))));
            }
            return FULL || piece * 16 < D ? counts : 0u;
        };
        // 16 codes of row i * STEP + my_row: two pieces of eight half-precision numbers
        auto store = [&](uint32_t to, uint4 (&w)[EACH], unsigned counts) {
            if (counts != (1u << EACH) - 1) {
#pragma unroll
                for (int i = 0; i < EACH; i++)
                    if (!((counts >> i) & 1)) w[i] = make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                const int row = i * STEP + my_row, c = 2 * piece;
                const uint32_t at = to + (c >> 3) * HALF_TILE + row * 128;
                uint32_t x[8];
                decode4<CODE>(w[i].x, x[0], x[1]);
                decode4<CODE>(w[i].y, x[2], x[3]);
                decode4<CODE>(w[i].z, x[4], x[5]);
                decode4<CODE>(w[i].w, x[6], x[7]);
                sts128(at + (((c & 7) ^ (row & 7)) << 4), x[0], x[1], x[2], x[3]);
                sts128(at + ((((c & 7) + 1) ^ (row & 7)) << 4), x[4], x[5], x[6], x[7]);
            }
        };
        // Values whose scale is not a power of two, as appending gives them: what is left of it, once more over what this thread has
        // stored, so that the ordinary way carries no test for it (in `store` it cost 5%, here 1.5%).
        auto multiply = [&](uint32_t to, unsigned odd, const float* rest) {
#pragma unroll 1
            for (int i = 0; i < 2 * EACH; i++) {
                const int row = (i >> 1) * STEP + my_row, c = 2 * piece;
                if (!((odd >> (row >> 4)) & 1)) continue;
                const uint32_t at = to + (c >> 3) * HALF_TILE + row * 128 + ((((c & 7) + (i & 1)) ^ (row & 7)) << 4);
                const __half2 f = __float2half2_rn(rest[row >> 4]);
                uint32_t x[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x[e]), f);
                    x[e] = *reinterpret_cast<const uint32_t*>(&y);
                }
                sts128(at, x[0], x[1], x[2], x[3]);
            }
        };
        uint4 kw[EACH], vw[EACH];
        if (p < 32) {
            ask_pages(0);
            ask_scales();
            note(0);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        unsigned k_counts = load(a.k, 0, kw), v_counts = load(a.v, 0, vw);
        for (int it = 0; it < n_it; it++) {
            const int stage = it % STAGES;
            const int next = (it & ~3) + 4;                          // the four tiles after these
            if (next < n_it) {
                if (p < 32) {
                    if ((it & 3) == 0) ask_pages(next);
                    if ((it & 3) == 1) ask_scales();
                    if ((it & 3) == 2) note(next);
                }
                if ((it & 3) == 2) asm volatile("bar.sync 1, 128;" ::: "memory");      // the producers: they have been noted
            }
            if (it >= STAGES) wait_for(&k_empty[stage], (it / STAGES - 1) & 1);
            store(base + OFF_K + stage * KV_BYTES, kw, k_counts);
            fence_async_proxy();
            // K of tile it is what the products after tile it - 1's weights wait for, V what those after its own do
            if (it == 0) {
                warp_arrive(&first_k);
            } else {
                warp_arrive(&go[0][(it - 1) & 1]);
                if (groups == 2) warp_arrive(&go[1][(it - 1) & 1]);
            }
            k_counts = load(a.k, it + 1, kw);
            if (it >= STAGES) wait_for(&v_empty[stage], (it / STAGES - 1) & 1);
            store(base + OFF_V + stage * KV_BYTES, vw, v_counts);
            const unsigned odd = s_runs[it % CONSTS] >> 8;
            if (odd) multiply(base + OFF_V + stage * KV_BYTES, odd, s_rest[it % CONSTS]);
            fence_async_proxy();
            for (int g = 0; g < groups; g++) {
                warp_arrive(&go[g][it & 1]);
                if (it == n_it - 1) warp_arrive(&go[g][it & 1]);     // there is no next K
            }
            v_counts = load(a.v, it + 1, vw);
        }
    } else {
        if (tid == ISSUE_WARP * 32 && n_it > 0) {
            // ---- products ------------------------------------------------------------------------------------------------------
            auto issue_s = [&](int g, int stage) {
                const uint32_t q = base + g * Q_BYTES, k = base + OFF_K + stage * KV_BYTES;
#pragma unroll
                for (int ks = 0; ks < HD / UMMA_K; ks++) {
                    const uint32_t off = (ks >> 2) * HALF_TILE + (ks & 3) * 32;
                    umma_bf16(tmem + s_col(g), make_smem_desc(q + off), make_smem_desc(k + off), IDESC_S, ks > 0);
                }
            };
            auto issue_pv = [&](int g, int stage, bool first_tile) {
                const uint32_t v = base + OFF_V + stage * KV_BYTES;
#pragma unroll
                for (int ks = 0; ks < BN / UMMA_K; ks++) {
                    // 16 keys are 2,048 bytes further; the second run of 64 dims is HALF_TILE behind the first (the leading byte offset)
                    uint64_t desc = make_smem_desc(v + ks * (UMMA_K * 128));
                    if (SUBS == 2) desc = (desc & ~((uint64_t)0x3fff << 16)) | ((uint64_t)(HALF_TILE >> 4) << 16);
                    umma_ta(tmem + o_col(g), tmem + s_col(g) + ks * (UMMA_K / 2), desc, IDESC_PV, !first_tile || ks > 0);
                }
            };
            wait_for(&first_k, 0);
            for (int g = 0; g < groups; g++) {
                wait_for(&q_ready[g], 0);
                tc_fence_after();
                issue_s(g, 0);
                umma_commit(&s_full[g]);
            }
            umma_commit(&k_empty[0]);
            for (int it = 0; it < n_it; it++) {
                const bool more = it + 1 < n_it;
                for (int g = 0; g < groups; g++) {
                    // one wait for all that the products need: each costs some 300 cycles, even when it is over
                    wait_for(&go[g][it & 1], (it >> 1) & 1);
                    tc_fence_after();
                    issue_pv(g, it % STAGES, it == 0);
                    if (g == groups - 1) umma_commit(&v_empty[it % STAGES]);
                    if (more) {
                        issue_s(g, (it + 1) % STAGES);
                        umma_commit(&s_full[g]);
                    } else {
                        umma_commit(&o_full[g]);
                    }
                }
                if (more) umma_commit(&k_empty[(it + 1) % STAGES]);
            }
        }
        __syncwarp();
    }
    if constexpr (SPLIT) {
        // ---- the cluster's sums, joined in its blocks' order: each block does its share of the rows, a row in a.splits pieces ------------
        const cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int rows = 256 / a.splits, row = rank * rows + (tid & (rows - 1)), width = HD / a.splits, d0 = tid / rows * width;
        if (tid < 256 && row < n_valid) {
            const int token = (first + row) / a.group, h = kvh * a.group + (first + row - token * a.group);
            const float4* sums = reinterpret_cast<const float4*>(smem_raw + (base - smem_u32(smem_raw)) + OFF_K);
            float m = -INFINITY, L = 0.0f;
            for (int k = 0; k < a.splits; k++) m = fmaxf(m, cluster.map_shared_rank(s_ml, k)[row].x);
            // a block that saw no key has no maximum and nothing to add; what is NaN has no maximum either, and counts
            auto factor_of = [&](float2 ml) { return ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ex2(ml.x - m); };
            for (int k = 0; k < a.splits; k++) {
                const float2 ml = cluster.map_shared_rank(s_ml, k)[row];
                L = fmaf(ml.y, factor_of(ml), L);
            }
            if (a.sink && m > -INFINITY) L += ex2(fmaf(a.sink[h], LOG2E, -m));
            float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;        // no visible key: zeros
            if (a.out_gate) inv *= a.out_gate[(size_t)(row0 + token) * a.n_heads + h];
            bf16* dst = a.out + (size_t)(row0 + token) * a.ld_out + (size_t)h * D;
            for (int d = d0; d < (FULL ? d0 + width : min(d0 + width, D)); d += 8) {
                float y[8] = {};
                for (int k = 0; k < a.splits; k++) {
                    const float f = factor_of(cluster.map_shared_rank(s_ml, k)[row]);
                    if (f == 0.0f) continue;
                    const float4* from = cluster.map_shared_rank(sums, k);
                    const float4 u = from[d / 4 * 256 + row], v = from[(d / 4 + 1) * 256 + row];
                    const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = fmaf(x[i], f, y[i]);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] *= inv;
                if (a.elem_gate) {
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] *= elem_gate_of(a.elem_gate, a.ld_elem_gate, a.gate_dim, row0 + token, h, d + i);
                }
                *reinterpret_cast<uint4*>(dst + d) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
            }
        }
        cluster.sync();                                              // no block leaves while another reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == ISSUE_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int CODE, int HD, bool FULL, bool SPLIT>
int launch(const Args& a, int n_seqs, long long tiles, cudaStream_t stream) {
    constexpr int SMEM = (2 + 2 * STAGES) * (HD / 64) * (int)HALF_TILE + 1024;
    static std::atomic<unsigned long long> told{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const unsigned long long bit = 1ull << (device & 63);
    if (!(told.load() & bit) || device > 63) {
        e = cudaFuncSetAttribute(prefill_8bit_kernel<CODE, HD, FULL, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return (int)e;
        told.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_kv_heads * a.splits, n_seqs, (unsigned)tiles);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (SPLIT) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = a.splits;
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
    e = cudaLaunchKernelEx(&cfg, prefill_8bit_kernel<CODE, HD, FULL, SPLIT>, a);
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

// Prompt portions as sandy_attention_8bit (attention_8bit.cu) takes them; num_splits 1, 2, 4 or 8 blocks share a block of rows' keys as a cluster,
// 0: the choice below.  bfloat16, heads of up to 128, pages of a multiple
// of 16 keys, rows of q and out on 16 bytes, a positive scale, no bias by distance, no cap above 512; SANDY_ERR_UNSUPPORTED for everything else, which the
// other kernel takes.
SANDY_API int sandy_prefill_attention_8bit_tc(const SandyAttend8* r, cudaStream_t stream) {
    if (!r) return SANDY_ERR_ARGUMENT;
    const SandyCache8& c = r->cache;
    const SandyAttentionRules& rules = r->rules;
    if (r->n_z == 0 || r->max_n == 0) return SANDY_OK;
    if (!r->q || !r->out || !r->positions || !r->q_start || !c.k || !c.v || !c.k_scale || !c.v_scale || !c.block_table || r->n_z < 0 ||
        r->max_n < 0 || c.max_blocks < 1 || c.page_size < 1)
        return SANDY_ERR_ARGUMENT;
    // a cap multiplies tanh_fast's 2^-22: at 512 a score is off by 2^-12.5 in units of log 2, less than its weight's rounding.  With the other
    // kernel's tanh_capped here, portions without a cap took 1.3% longer too, those with one 4%.
    if (rules.softcap > 512.0f) return SANDY_ERR_UNSUPPORTED;
    if (c.dtype != SANDY_BF16 || rules.dist_bias || rules.window < 0 || rules.keep_first < 0 || rules.chunk < 0 || !(rules.softcap >= 0.0f) ||
        (rules.keep_first > 0 && rules.chunk > 0) || (rules.elem_gate && rules.gate_dim < 1) || !(r->scale > 0.0f))
        return SANDY_ERR_UNSUPPORTED;
    if (c.head_dim < 16 || c.head_dim > 128 || c.head_dim % 16 || c.page_size % 16 || c.n_kv_heads < 1 || r->n_heads % c.n_kv_heads) return SANDY_ERR_UNSUPPORTED;
    if (c.page_stride % 16 || (((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)r->q | (uintptr_t)r->out) & 15) || r->ld_q % 8 || r->ld_out % 8 ||
        r->n_z > 65535 || r->num_splits < 0 || r->num_splits > 8 || (r->num_splits & (r->num_splits - 1)) || (long long)r->max_n * (r->n_heads / c.n_kv_heads) > 65535 * 256ll)
        return SANDY_ERR_UNSUPPORTED;
    Args a = {};
    a.q = (const bf16*)r->q;
    a.k = (const uint8_t*)c.k;
    a.v = (const uint8_t*)c.v;
    a.k_scale = c.k_scale;
    a.v_scale = c.v_scale;
    a.block_table = c.block_table;
    a.q_start = r->q_start;
    a.kv_before = r->positions;
    a.out = (bf16*)r->out;
    a.status = c.status;
    a.sink = rules.sink;
    a.out_gate = rules.out_gate;
    a.elem_gate = (const bf16*)rules.elem_gate;
    a.ld_q = r->ld_q;
    a.ld_out = r->ld_out;
    a.page_stride = c.page_stride;
    a.scale_stride = c.scale_stride;
    a.max_blocks = c.max_blocks;
    a.n_rows = r->n_rows;
    a.max_n = r->max_n;
    a.n_heads = r->n_heads;
    a.n_kv_heads = c.n_kv_heads;
    a.group = r->n_heads / c.n_kv_heads;
    a.page_size = c.page_size;
    a.page_shift = (c.page_size & (c.page_size - 1)) == 0 ? __builtin_ctz(c.page_size) : -1;
    a.num_pages = c.num_pages;
    a.head_dim = c.head_dim;
    a.window = rules.window;
    a.keep_first = rules.keep_first;
    a.chunk = rules.chunk;
    a.ld_elem_gate = rules.ld_elem_gate;
    a.gate_dim = rules.gate_dim;
    a.scale = r->scale;
    a.softcap = rules.softcap;
    const long long tiles = ((long long)r->max_n * a.group + 255) / 256, blocks = tiles * c.n_kv_heads * r->n_z;
    a.splits = r->num_splits;
    if (!a.splits) {
        // As many blocks as fit the SMs at once, each with a key tile at least.  256 tokens behind 6,000, 32 heads of 128 on 8: one block
        // for all keys 135 us, two 80, four 51, eight (two rounds) 112; behind 20,000, 8 heads: 430, 228, 125, 75; a prompt of 950
        // tokens, 12 heads of 64: 27, 20, 33, 65.
        a.splits = 1;
        while (a.splits < 8 && blocks * a.splits * 2 <= sandy_sm_count() && r->max_keys >= a.splits * 2 * BN) a.splits *= 2;
    }
#define LAUNCH(CODE, HD, FULL) \
    return a.splits > 1 ? launch<CODE, HD, FULL, true>(a, r->n_z, tiles, stream) : launch<CODE, HD, FULL, false>(a, r->n_z, tiles, stream)
#define SIZES(CODE)                                         \
    do {                                                    \
        if (c.head_dim == 64) LAUNCH(CODE, 64, true);       \
        if (c.head_dim == 128) LAUNCH(CODE, 128, true);     \
        if (c.head_dim < 64) LAUNCH(CODE, 64, false);       \
        LAUNCH(CODE, 128, false);                           \
    } while (0)
    if (c.code == SANDY_E4M3) SIZES(SANDY_E4M3);
    if (c.code == SANDY_INT8) SIZES(SANDY_INT8);
#undef SIZES
#undef LAUNCH
    return SANDY_ERR_UNSUPPORTED;
}
