// Causal attention over the paged cache in 8 bits (kv_8bit.cuh), of single tokens and of prompt portions.
//
// Formula: attention.cu's, with keys ck_j * sk and values cv_j * sv, sk and sv the scales of key j's block, and the rules of
// attention_rules.h.  Head sizes: multiples of 16 up to 256.
//
// Layout.  The queries that read one key/value head of one request -- the heads of its group, and in a prompt portion the
// portion's tokens -- are the COLUMNS of the products, keys and value dimensions the rows:
//   S [16 keys x 8 queries]   = codes of K [16 x 16 dims] x q [16 dims x 8]       mma.sync m16n8k16, half precision, float sums
//   O [16 dims x 8 queries]  += codes of V^T [16 dims x 16 keys] x P [16 keys x 8]
// The codes are the wide operand, so an instruction takes in 256 of them however few queries there are (one to eight heads in a
// group), and what the conversion costs (one cvt for two e4m3 codes, five operations for four int8 codes) is paid once for all
// columns.  The order of dims inside the first product and of keys inside the second is free; it is chosen so that a lane's
// operands are pieces of rows as they lie in the cache: for K 16 consecutive dims of keys g and g + 8 (g = lane / 4), for V
// consecutive dims of keys 2t, 2t+1, 2t+8, 2t+9 (t = lane % 4), whose bytes are paired by a byte permutation.  S comes out with keys in
// the lane groups; movmatrix turns P, as half-precision pairs, into the operand of the second product.
//
// A warp walks keys of its own: it copies them (cp.async, 16 bytes a lane) into a ring of three stages that no other warp touches, so
// that there is no barrier before the end.  A row's pieces are exchanged and a tile's keys are taken in an order by which a
// quarter warp's reads of keys and half a warp's of values meet all banks.  Pages and scales of the next 16 tiles are looked up at
// once, a run of keys a lane, so that the chain from the block table over the scale to the copy is not walked for every tile.
//
// Scales.  A score is S * sk * (2^eq * scale), a factor a key.  A value's scale joins the weight: with x_j = s_j + log2(sv_j) (s in units of
// log 2) and a reference M near the largest x so far, 2^(x_j - M) / sv_j is summed for the denominator and 2^(x_j - M) is rounded to
// half precision for the product.  No block's values are out of half precision's range this way.
// M moves to HEADROOM = 7 below the largest x, and only when an x is above M + RESCALE = 14: weights stay below 2^14 (2^15 where a scale is no
// power of two), and what is 2^-32 of the largest still rounds to something.  With the largest at 1, all of e^-18 and
// below was nothing: 100,000 such keys were missing in the result, though not in the denominator.
//
// Roundings.  q is scaled by a power of two (2^eq) so that its largest element lies in [1, 2) and rounded to half precision:
// exact for bfloat16 elements above 2^-14 of the largest, off by 2^-25 of it at most.  P rounds to 11 bits, the row sum is taken
// before.  For float32 both are split into two half-precision pieces (22 bits), which lie in neighbouring columns; the two
// columns' results are in the same lane and are added there.  The second piece is held times 2^11 (SECOND), so that it has its 11 bits
// wherever the first has one: a number is off by 2^-22 of itself or 2^-36 of the largest, whichever is more.  At its own size it would end
// where half precision does, at 2^-25 of the largest, and a hundred thousand weights of e^-18 beside one of 1 were missing in
// the result, though not in the denominator.
//
// What bounds it.  Single tokens: the codes' bytes.  16 warps an SM (in blocks of four, or two where there are very many) with
// three stages of 4 KB each keep 190 KB on their way.  Where there are few requests `num_splits` blocks share one's keys: up to 8 are a
// cluster, whose first block takes the others' results over its shared memory; more leave theirs in scratch, which a second kernel joins
// in a fixed order.  Measured (bfloat16): 8 tokens x 12 heads of 64 behind 100 to 900 keys (e4m3) 6.9 us, of which half is the launch, the
// lookup and the join; 64 x 25 heads behind 64 to 1,000 (int8) 32.8 us, 3.2 TB/s of codes: 13 us with 64 keys each, what a block's
// beginning and end cost in 2.7 rounds; behind 8,000 keys each 266 us, 94% of 6.57 TB/s; 4 requests of 8 heads of 128 (e4m3), each read by 4,
// behind 30,000 to 100,000 keys 120 us, 80% (a call by itself 127: two kernels).  These are tables as wide as the longest request: splits are
// cut from the table's width, so that a request much shorter than its table is walked by the first of them.
// Where a key/value head has one query head, bfloat16 kernels keep one column a lane instead of two (ONE): a tenth fewer instructions, 32.4 us
// instead of 36.9 above.
// Prompt portions: the tensor cores' warp-level instructions; the tcgen05 kernel takes over from 33 query rows on where it can.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "cache8.h"
#include "kv_8bit.cuh"

static_assert(sizeof(SandyAttend8) == 256, "the layout callers lay down");

namespace cg = cooperative_groups;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float SECOND = 2048.0f;        // what the second piece of a float32 number is multiplied by
constexpr float FAR = 8388608.0f;        // 2^23: the largest score, in units of log 2, under a cap or a bias
constexpr int FOLD = 32;                 // groups of keys that a float32 warp sums by themselves

struct Args {
    const void* q;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const int *block_table, *token_seq, *positions, *q_start;       // q_start: prompt portions (positions: kv_before), else single tokens
    void* out;
    float* scratch;                                                  // partial results, with num_splits > 1
    int* status;
    const float *sink, *out_gate, *dist_bias;
    const void* elem_gate;
    long long ld_q, ld_out, page_stride, scale_stride;
    int max_blocks, n_rows, max_n, n_seqs, n_heads, n_kv_heads, head_dim, page_size, num_pages, num_splits, split_tiles, group, page_shift;    // heads of a key/value head; -1: no power of two
    int window, keep_first, chunk, n_dist, ld_elem_gate, gate_dim;
    float scale, softcap;
    bool two_warps;                                                  // blocks of two warps instead of four
    bool in_cluster;                                                 // the splits of a block of queries are a cluster
    bool q_aligned;                                                  // q's rows start on 16 bytes
};

__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of half-precision numbers, two of a row in a lane, turned
__device__ __forceinline__ unsigned turn(unsigned x) {
    unsigned y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float max_over_groups(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// Sixteen elements as floats, zeros where they are not there.
template <typename T>
__device__ __forceinline__ void load16(const T* __restrict__ p, bool there, bool aligned, float (&x)[16]) {
    if (!there) {
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = 0.0f;
    } else if (!aligned) {
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = to_f32(p[e]);
    } else if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 v = reinterpret_cast<const float4*>(p)[i];
            x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[8 * i + 2 * e] = __uint_as_float(w[e] << 16);
                x[8 * i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    }
}

// Where a block's queries stand: `n` new tokens from row `row0` on, the first at position `before` of request `seq`.
struct Portion {
    int seq, row0, n, before;
};
__device__ __forceinline__ Portion portion_of(const Args& a, int z) {
    Portion p;
    p.seq = a.q_start ? z : a.token_seq[z];
    p.row0 = a.q_start ? a.q_start[z] : z;
    p.n = a.q_start ? a.q_start[z + 1] - p.row0 : 1;
    p.before = a.positions[z];
    // rows that are not there, or no block is there for, or whose positions are no int
    if (p.row0 < 0 || p.n > a.n_rows - p.row0 || p.n > a.max_n || (long long)p.before + p.n - 1 > 0x7fffffffll) {
        if (p.n > 0 && a.status && threadIdx.x == 0) atomicOr(a.status, 16);
        p.n = 0;
    }
    return p;
}

// The first visible key of a query behind its kept ones.
__device__ __forceinline__ int first_key(const Args& a, int pos) {
    int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    if (a.chunk > 0) lo = max(lo, pos - pos % a.chunk);
    return lo;
}

// A head's result, its sum of weights and the maximum they refer to, as an output element.
template <typename T>
__device__ __forceinline__ void finish(const Args& a, float O, float L, float M, int row, int h, int d) {
    if (a.sink && M > -INFINITY) L += ex2(fmaf(a.sink[h], LOG2E, -M));
    float y = L > 0.0f || L != L ? O / L : 0.0f;                     // no visible key: zero
    if (a.out_gate) y *= a.out_gate[(size_t)row * a.n_heads + h];
    y *= elem_gate_of((const T*)a.elem_gate, a.ld_elem_gate, a.gate_dim, row, h, d);
    ((T*)a.out)[(size_t)row * a.ld_out + (size_t)h * a.head_dim + d] = from_f32<T>(y);
}

constexpr float RESCALE = 14.0f;         // how far (in the exponent) a score may be above the reference of its column
constexpr float HEADROOM = 7.0f;         // how far below the largest score the reference is set

// What a warp has looked up about a run of keys in one page: where its rows start (page 0's, if it has no page), its block's scales
// and what is made of them: ev = log2 of the value's scale, inv = 2^-ev.
struct __align__(16) Run {
    long long off;                       // what copying reads
    unsigned flags;
    float vs;
    float ks, ev, inv;                   // what the products read
    unsigned again;                      // the flags once more
};
constexpr unsigned HAS_PAGE = 1;         // there is a page
constexpr unsigned NO_POWER = 2;         // vs is not 2^ev: the weights are multiplied by it
constexpr unsigned SEEN_BY_ALL = 4;      // every query of the block sees all keys of the tile, and scores are as they are
constexpr unsigned SEEN_BY_ONE = 8;      // every key of the tile is seen by one query or more

// Stages of KT tiles of 16 keys that a warp has on their way: 12 KB at heads of 64 with two tiles a stage and at heads of 128 with one, 24 KB at
// heads of 256, 6 KB at heads of 64 with one (odd pages, and blocks of 32 columns).
constexpr int STAGES = 3;

// Where piece p (16 bytes) of row r lies in its row: what a quarter warp reads at a time of the keys (two rows' 64 bytes) and half
// a warp of the values (four rows' 32 bytes) then comes from different banks.
template <int DMAX>
__device__ __forceinline__ int swizzled(int r, int p) {
    return DMAX == 64 ? p ^ (r & 2) : p ^ (2 * (r & 3));
}
// Which key of a tile's first eight is row g of the first product, for the same reason: 0, 7, 1, 6, 2, 5, 3, 4.
__device__ __forceinline__ int row_key(int g) { return g & 1 ? 7 - (g >> 1) : g >> 1; }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void lds128(unsigned (&w)[4], uint32_t at) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void lds64(unsigned (&w)[2], uint32_t at) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
}

// ev and inv of a value's scale: log2 of it, but at least -60.  With the 2^-100 of a block of zeros in the reference, weights beside blocks
// of large values would run out of float's exponents, and be missing in the denominator.  Of a scale that is not finite ev = 0, so
// that its weights are NaN and the others stay numbers.
__device__ __forceinline__ unsigned power_of(float vs, float& ev, float& inv) {
    const unsigned bits = __float_as_uint(vs);
    const int biased = (int)(bits >> 23) & 255, e = biased == 255 ? 127 : max(biased, 127 - 60);
    ev = (float)(e - 127);
    inv = __uint_as_float((unsigned)max(254 - e, 0) << 23);
    return bits != (unsigned)e << 23 || biased == 255 ? NO_POWER : 0u;
}

// WARPS: of a block; DMAX: 64, 128 or 256, the head size rounded up; DK: the head size, or 0 where it is known at run time only; NT: column tiles of
// 8; KT: key tiles of 16 that a warp takes at a time; RUN: 16 or 8, pages are a multiple of it, so that a tile or half a tile lies in
// one page; 0: every row is looked up by itself.  ONE: a block has one query, in column 0.
template <typename T, int CODE, int WARPS, int DMAX, int DK, int NT, int KT, int RUN, bool ONE = false>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 && DMAX < 256 ? 16 / WARPS : 1)
attention_8bit_kernel(const __grid_constant__ Args a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;            // pieces a number is split into
    constexpr int QT = 8 * NT / P;                       // queries of a block
    constexpr int CH = DMAX / 64;                        // runs of 64 dims
    constexpr int Q2 = P == 2 || ONE ? 1 : 2;                            // queries in a lane's two columns of a tile
    constexpr int STAGE = 2 * KT * 16 * DMAX;
    // a warp's stages [STAGES][keys | values][KT * 16 rows of DMAX bytes]; at the end the warps' sums in the same place
    extern __shared__ __align__(128) uint8_t smem[];
    float (*sm_o)[QT][DMAX + 1] = reinterpret_cast<float (*)[QT][DMAX + 1]>(smem);
    __shared__ float sm_m[WARPS][QT], sm_l[WARPS][QT];
    constexpr int HALVES = RUN == 16 ? 1 : 2;            // runs of a tile
    constexpr int BATCH = 16 / HALVES;                   // tiles a warp looks up at a time; it keeps two batches
    __shared__ Run known[RUN ? WARPS : 1][RUN ? 32 : 1];

    pdl_launch_dependents();
    pdl_wait();
    const int z = blockIdx.z, kvh = blockIdx.y;
    const int tile = a.num_splits == 1 ? blockIdx.x : blockIdx.x / a.num_splits, split = blockIdx.x - tile * a.num_splits;
    const Portion at = portion_of(a, z);
    const int group = a.group;
    const int n_queries = min(QT, at.n * group - tile * QT);         // of this block
    if (n_queries <= 0) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int D = DK ? DK : a.head_dim, ps = a.page_size;
    // query qi of the (request, key/value head): which of its tokens, which head of the group
    const bool single = !a.q_start || group == 1;
    auto token_of = [&](int qi) { return a.q_start ? single ? qi : qi / group : 0; };
    auto head_of = [&](int qi) { return kvh * group + (a.q_start ? single ? 0 : qi % group : qi); };

    const bool plain = a.softcap == 0.0f && !a.dist_bias;            // a score is S times its factors
    // ---- the block's keys, as tiles of 16 positions: kept first ones, then from the first query's first to the last query's own ----
    const int pos_first = at.before + token_of(tile * QT), pos_last = at.before + token_of(tile * QT + n_queries - 1);
    const int lo_first = first_key(a, max(pos_first, 0)), lo_last = first_key(a, max(pos_last, 0));
    // positions behind the block table's end have no page: no tile is walked for them, however far they are
    const long long in_table = (long long)a.max_blocks * ps;
    const int key_last = (int)min((long long)pos_last, in_table - 1);
    const int kept_tiles = lo_first > 0 ? min((int)((min((long long)a.keep_first, in_table) + 15) >> 4), lo_first >> 4) : 0;
    const bool request = (unsigned)at.seq < (unsigned)a.n_seqs;
    if ((!request || key_last < pos_last) && tid == 0 && a.status) atomicOr(a.status, 16);
    const int n_tiles = request && pos_last >= 0 ? kept_tiles + max((key_last >> 4) - (lo_first >> 4) + 1, 0) : 0;
    const int tile_end = split == a.num_splits - 1 ? n_tiles : min(n_tiles, (split + 1) * a.split_tiles);
    const int* table = a.block_table + (size_t)(request ? at.seq : 0) * a.max_blocks;
    const size_t head_at = (size_t)kvh * ps * D;
    auto seen = [&](int j) { return j <= pos_last && (j >= lo_first || j < a.keep_first); };      // by any of the block's queries

    float o[CH * 4][NT][4];
    float M[NT][Q2], l[NT][Q2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int j = 0; j < CH * 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[j][n][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < Q2; e++) {
            M[n][e] = -INFINITY;
            l[n][e] = 0.0f;
        }
    }

    // This warp's tiles: KT at a time, the first at `tile0`, then every WARPS * KT-th group.
    const int tile0 = split * a.split_tiles + warp * KT;
    const int n_groups = tile0 < tile_end ? (tile_end - tile0 + WARPS * KT - 1) / (WARPS * KT) : 0;
    auto nth_of = [&](int group_at, int kt) { return tile0 + group_at * WARPS * KT + kt; };
    auto first_of = [&](int nth) { return (nth < kept_tiles ? nth : nth - kept_tiles + (lo_first >> 4)) << 4; };

    // pages and scales of the next BATCH tiles, a run a lane, for all lanes to read; the batch before stays
    auto look_up = [&](int group_at) {
        __syncwarp();
        const int in = group_at * KT + lane / HALVES, half = lane % HALVES;
        const int nth = nth_of(in / KT, in % KT), key0 = first_of(nth), j = key0 + 8 * half;
        Run run = {};
        run.flags = (key0 + 15 <= pos_first && key0 >= lo_last && plain ? SEEN_BY_ALL : 0) |
                    (key0 + 15 <= pos_last && key0 >= lo_first ? SEEN_BY_ONE : 0);
        if (lane < 16 && nth < tile_end && j <= pos_last && (j + RUN - 1 >= lo_first || j < a.keep_first)) {
            const int b = a.page_shift >= 0 ? j >> a.page_shift : j / ps;
            const int page = b < a.max_blocks ? table[b] : -1;
            if (page >= 0 && page < a.num_pages) {
                run.off = page * a.page_stride + (long long)(head_at + (size_t)(j - b * ps) * D);
                run.ks = a.k_scale[page * a.scale_stride + kvh];
                run.vs = a.v_scale[page * a.scale_stride + kvh];
                run.flags |= HAS_PAGE | power_of(run.vs, run.ev, run.inv);
            } else if (a.status) {
                atomicOr(a.status, 16);
            }
        }
        run.again = run.flags;
        if (lane < 16) known[warp][(HALVES * in + half) % 32] = run;
        __syncwarp();
    };
    // RUN 0: the row of key j, if a query sees it and it has a page
    auto row_of = [&](int nth, int j, size_t& off, int& page) {
        if (nth >= tile_end || !seen(j)) return false;
        const int b = j / ps;
        page = b < a.max_blocks ? table[b] : -1;
        if (page < 0 || page >= a.num_pages) {
            if (a.status) atomicOr(a.status, 16);
            return false;
        }
        off = (size_t)page * a.page_stride + head_at + (size_t)(j - b * ps) * D;
        return true;
    };

    // Copies a group's rows, 16 bytes a lane, into its stage; rows that no query sees, and those without a page, become zeros (a
    // weight of 0 times what such a row may hold would be NaN).  Piece p of row r lies at piece swizzled(r, p).
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * STAGES * STAGE;
    constexpr int PIECES = DMAX / 16, STEP = 32 / PIECES;            // of a row; rows that a warp copies at a time
    const int my_piece = lane % PIECES, my_row = lane / PIECES;
    const uint32_t my_place = my_row * DMAX + swizzled<DMAX>(my_row, my_piece) * 16;      // of rows my_row + a multiple of 4
    const uint8_t *my_k = a.k + (my_row * D + my_piece * 16), *my_v = a.v + (my_row * D + my_piece * 16);
    auto copy = [&](int group_at, int stage) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            const uint32_t to = ring + stage * STAGE + kt * 16 * DMAX;
            if constexpr (RUN == 16) {
                const uint4 run = *reinterpret_cast<const uint4*>(&known[warp][(group_at * KT + kt) % 32]);
                if ((run.z & (HAS_PAGE | SEEN_BY_ONE)) == (HAS_PAGE | SEEN_BY_ONE)) {          // all of the tile, as it lies
                    const long long off = (long long)((unsigned long long)run.y << 32 | run.x);
                    const uint8_t *k = my_k + off, *v = my_v + off;
#pragma unroll
                    for (int i = 0; i < 16 / STEP; i++) {
                        copy16(to + my_place + i * STEP * DMAX, k + i * STEP * D);
                        copy16(to + my_place + i * STEP * DMAX + KT * 16 * DMAX, v + i * STEP * D);
                    }
                    continue;
                }
            }
            const int nth = nth_of(group_at, kt), key0 = first_of(nth);
#pragma unroll
            for (int i = 0; i < 16 / STEP; i++) {
                const int row = i * STEP + my_row;
                size_t off = 0;
                bool ok;
                if constexpr (RUN != 0) {
                    const Run& run = known[warp][(HALVES * (group_at * KT + kt) + (RUN == 16 ? 0 : row >> 3)) % 32];
                    off = run.off + (size_t)(RUN == 16 ? row : row & 7) * D;
                    ok = (run.flags & HAS_PAGE) && ((run.flags & SEEN_BY_ONE) || seen(key0 + row));
                } else {
                    int page = 0;
                    ok = row_of(nth, key0 + row, off, page);
                }
                if (!DK) ok = ok && my_piece * 16 < D;               // dims there are not: zeros too
                const uint32_t dst = to + row * DMAX + swizzled<DMAX>(row, my_piece) * 16;
                copy16(dst, a.k + off + my_piece * 16, ok);
                copy16(dst + KT * 16 * DMAX, a.v + off + my_piece * 16, ok);
            }
        }
    };

    if (RUN != 0 && n_groups > 0) look_up(0);
#pragma unroll
    for (int st = 0; st < STAGES; st++) {
        if (st < n_groups) copy(st, st);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // ---- q: column g of every tile, as the second operand ------------------------------------------------------
    unsigned qf[NT][CH * 4][2];
    float my_factor[NT];                                 // of column g
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int i = (n * 8 + g) / P, qi = tile * QT + (i < n_queries ? i : 0);
        const T* src = (const T*)a.q + (size_t)(at.row0 + token_of(qi)) * a.ld_q + (size_t)head_of(qi) * D;
        float x[CH][16];                                 // dims 64 c + 16 t ..
        unsigned amax = 0;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            load16(src + 64 * c + 16 * t, i < n_queries && 64 * c + 16 * t < D, a.q_aligned, x[c]);
#pragma unroll
            for (int e = 0; e < 16; e++) amax = max(amax, __float_as_uint(x[c][e]) & 0x7fffffffu);
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e2 = max(-100, min(120, (int)(amax >> 23) - 127));
        const float down = __uint_as_float((unsigned)(127 - e2) << 23);
        my_factor[n] = __uint_as_float((unsigned)(127 + e2) << 23) * a.scale;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int w = 0; w < 8; w++) {                // word w: dims 64 c + 16 t + 2 w, + 1; k-step w / 2
                float x0 = x[c][2 * w] * down, x1 = x[c][2 * w + 1] * down;
                if (P == 2 && (g & 1)) {                 // the second piece: what the first one leaves
                    x0 = (x0 - __half2float(__float2half_rn(x0))) * SECOND;
                    x1 = (x1 - __half2float(__float2half_rn(x1))) * SECOND;
                }
                qf[n][c * 4 + (w >> 1)][w & 1] = pack_half(x0, x1);
            }
    }
    // the lane's two columns 2t, 2t + 1 of every tile: one query each, or the two pieces of one
    float factor[NT][Q2];                                // S times this and the key's scale: a score, in units of log 2 if `plain`
    int pos[NT][Q2], lo[NT][Q2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < Q2; e++) {
            const int i = (n * 8 + 2 * t) / P + e;
            factor[n][e] = __shfl_sync(0xffffffffu, my_factor[n], (2 * t + e) * 4) * (plain ? LOG2E : 1.0f);
            pos[n][e] = i < n_queries ? at.before + token_of(tile * QT + i) : -1;
            lo[n][e] = first_key(a, max(pos[n][e], 0));
        }

    // rows of the first product and columns of the second: key `my_key` (+ 8) of a tile for lane group g, see row_key()
    const int my_key = row_key(g);
    // float32: the sums of the groups before the last FOLD ones, and what they are to be multiplied by since.  The tensor cores cut what they
    // add to a sum, and do not round it: 100,000 keys in one split were off by 1.4e-4 of the largest value.  Costs 1 to 5%.
    float o_all[P == 2 ? CH * 4 : 1][NT][4], l_all[NT][Q2], since[NT][Q2];
    if (P == 2) {
#pragma unroll
        for (int n = 0; n < NT; n++) since[n][0] = 1.0f;
    }
    int stage = 0, it = 0;
    auto fold = [&]() {
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < (P == 2 ? CH * 4 : 1); j++)
#pragma unroll
                for (int e = 0; e < 4; e++) o_all[j][n][e] = it > FOLD ? fmaf(o_all[j][n][e], since[n][0], o[j][n][e]) : o[j][n][e];
            l_all[n][0] = it > FOLD ? fmaf(l_all[n][0], since[n][0], l[n][0]) : l[n][0];
        }
    };
    while (it < n_groups) {
        for (const int stop = P == 2 ? min(n_groups, it + FOLD) : n_groups; it < stop; it++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");      // group `it` has landed (a lane's own copies),
            __syncwarp();                                                                  // and every lane's
            const uint32_t k_at = ring + stage * STAGE, v_at = k_at + KT * 16 * DMAX;
            // of keys my_key and my_key + 8 (RUN 16: of both) of the group's tiles: scales and what is made of them, flags
            constexpr int R = RUN == 16 ? 1 : 2;
            float ks[KT][R], ev[KT][R], inv[KT][R], vs[KT][R];
            unsigned flags[KT][R];
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int r = 0; r < R; r++) {
                    if constexpr (RUN != 0) {
                        const float4 run = *reinterpret_cast<const float4*>(&known[warp][(HALVES * (it * KT + kt) + r) % 32].ks);
                        ks[kt][r] = run.x;
                        ev[kt][r] = run.y;
                        inv[kt][r] = run.z;
                        flags[kt][r] = __float_as_uint(run.w);
                    } else {
                        size_t off = 0;
                        int page = 0;
                        const bool ok = row_of(nth_of(it, kt), first_of(nth_of(it, kt)) + my_key + 8 * r, off, page);
                        ks[kt][r] = ok ? a.k_scale[(size_t)page * a.scale_stride + kvh] : 0.0f;
                        vs[kt][r] = ok ? a.v_scale[(size_t)page * a.scale_stride + kvh] : 0.0f;
                        flags[kt][r] = power_of(vs[kt][r], ev[kt][r], inv[kt][r]) | (ok ? HAS_PAGE : 0u);
                    }
                }

            auto vs_of = [&](int kt, int r) { return RUN != 0 ? known[warp][(HALVES * (it * KT + kt) + r) % 32].vs : vs[kt][r]; };
            unsigned every = HAS_PAGE | SEEN_BY_ALL, some = 0;          // flags that all of the group's keys have, that one has
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int r = 0; r < R; r++) {
                    every &= flags[kt][r];
                    some |= flags[kt][r];
                }
            const bool plainly = RUN && every == (HAS_PAGE | SEEN_BY_ALL);       // no mask, no rule

            // ---- S ----------------------------------------------------------------------------------------------------
            float sc[KT][NT][4];
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[kt][n][e] = 0.0f;
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    unsigned w0[4], w1[4];                    // 16 dims of keys my_key, my_key + 8
                    lds128(w0, k_at + (kt * 16 + my_key) * DMAX + swizzled<DMAX>(my_key, 4 * c + t) * 16);
                    lds128(w1, k_at + (kt * 16 + my_key + 8) * DMAX + swizzled<DMAX>(my_key, 4 * c + t) * 16);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        unsigned a0, a1, a2, a3;
                        decode4<CODE>(w0[i], a0, a2);
                        decode4<CODE>(w1[i], a1, a3);
#pragma unroll
                        for (int n = 0; n < NT; n++) mma_f16(sc[kt][n], a0, a1, a2, a3, qf[n][c * 4 + i][0], qf[n][c * 4 + i][1]);
                    }
                }
            }

            // ---- x = score + log2 of the value's scale, -inf where the key is not seen ------------------------------------
            float top[NT][Q2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Q2; e++) top[n][e] = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < Q2; e++) {
                            float x = P == 2 ? fmaf(sc[kt][n][2 * r + 1], 1.0f / SECOND, sc[kt][n][2 * r]) : sc[kt][n][2 * r + e];
                            if (plainly) {
                                x = fmaf(x, ks[kt][r % R] * factor[n][e], ev[kt][r % R]);
                            } else {
                                const int j = first_of(nth_of(it, kt)) + my_key + 8 * r;
                                const bool visible = (flags[kt][r % R] & HAS_PAGE) && j <= pos[n][e] && (j >= lo[n][e] || j < a.keep_first);
                                x *= ks[kt][r % R] * factor[n][e];
                                if (!plain) {
                                    if (a.softcap > 0.0f) x = a.softcap * (P == 2 ? tanhf(x / a.softcap) : tanh_capped(x / a.softcap));
                                    if (a.dist_bias && visible)
                                        x += a.dist_bias[(size_t)head_of(tile * QT + (n * 8 + 2 * t) / P + e) * a.n_dist + min(pos[n][e] - j, a.n_dist - 1)];
                                    // far below and above what softmax tells apart (a bias as a mask: -1e30, or the type's lowest number): whole
                                // numbers of x still add up with the value's log2 there, so that a row of such keys alone is their mean
                                const float y = x * LOG2E;
                                x = fabsf(y) > FAR && fabsf(x) < INFINITY ? copysignf(FAR, x) : y;
                                }
                                x = visible ? x + ev[kt][r % R] : -INFINITY;
                            }
                            sc[kt][n][P == 2 ? 2 * r : 2 * r + e] = x;
                            top[n][e] = fmaxf(top[n][e], x);
                        }
            }
            // The column's reference moves when a score has run far ahead of it (always on the first keys), for the whole warp together.
            bool move = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Q2; e++) move |= top[n][e] > M[n][e] + RESCALE;
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < Q2; e++) {
                        const float m = fmaxf(M[n][e], max_over_groups(top[n][e]) - HEADROOM);
                        const float shrink = m == -INFINITY ? 1.0f : ex2(M[n][e] - m);
                        M[n][e] = m;
                        l[n][e] *= shrink;
                        if (P == 2) since[n][e] *= shrink;
#pragma unroll
                        for (int j = 0; j < CH * 4; j++) {
                            o[j][n][e] *= shrink;
                            o[j][n][e + 2] *= shrink;
                            if (P == 2) {
                                o[j][n][1] *= shrink;
                                o[j][n][3] *= shrink;
                            }
                        }
                    }
            }
            float m_use[NT][Q2];                              // a column that has seen no key yet: its weights are 2^-inf
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Q2; e++) m_use[n][e] = M[n][e] == -INFINITY ? 0.0f : M[n][e];
            // ---- weights, as the second operand; O ---------------------------------------------------------------------
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
                unsigned pf[NT][2];
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        // 2^(x - M) is the weight times the value's scale, where that is a power of two: what appending gives
                        float w[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int e = 0; e < Q2; e++) {
                            const float x = sc[kt][n][P == 2 ? 2 * r : 2 * r + e];
                            w[e] = ex2(x - m_use[n][e]);
                            l[n][e] = fmaf(w[e], inv[kt][r % R], l[n][e]);
                            if (some & NO_POWER) w[e] = x == -INFINITY ? 0.0f : w[e] * inv[kt][r % R] * vs_of(kt, r % R);
                        }
                        if (P == 2) w[1] = (w[0] - __half2float(__float2half_rn(w[0]))) * SECOND;
                        pf[n][r] = turn(pack_half(w[0], w[1]));
                    }
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    unsigned vw[4][2];                        // dims 64 c + 8 g .. of the keys of the second product's columns 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int low = r & 1 ? 7 - t : t, row = low + 8 * (r >> 1);
                        lds64(vw[r], v_at + (kt * 16 + row) * DMAX + swizzled<DMAX>(low, 4 * c + (g >> 1)) * 16 + (g & 1) * 8);
                    }
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        unsigned w[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) w[r] = vw[r][half];
                        // bytes of two keys side by side: dims d, d + 1 and d + 2, d + 3 of the piece's four
                        const unsigned e0 = __byte_perm(w[0], w[1], 0x5140), e1 = __byte_perm(w[0], w[1], 0x7362);
                        const unsigned f0 = __byte_perm(w[2], w[3], 0x5140), f1 = __byte_perm(w[2], w[3], 0x7362);
                        unsigned a0, a1, a2, a3;
                        decode4<CODE>(e0, a0, a1);
                        decode4<CODE>(f0, a2, a3);
#pragma unroll
                        for (int n = 0; n < NT; n++) mma_f16(o[c * 4 + half * 2][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                        decode4<CODE>(e1, a0, a1);
                        decode4<CODE>(f1, a2, a3);
#pragma unroll
                        for (int n = 0; n < NT; n++) mma_f16(o[c * 4 + half * 2 + 1][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                    }
                }
            }
            __syncwarp();                                     // the stage may be written again
            if (it + STAGES < n_groups) {
                if constexpr (RUN != 0)
                    if ((it + STAGES) * KT % BATCH == 0) look_up(it + STAGES);
                copy(it + STAGES, stage);
            }
            stage = stage == STAGES - 1 ? 0 : stage + 1;
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        if (P == 2 && n_groups > FOLD) {
            fold();
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int j = 0; j < CH * 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[j][n][e] = it < n_groups ? 0.0f : o_all[P == 2 ? j : 0][n][e];
                l[n][0] = it < n_groups ? 0.0f : l_all[n][0];
                since[n][0] = 1.0f;
            }
        }
    }
    __syncthreads();                                      // no stage is in use any more
    if (a.in_cluster) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    // ---- the warps' states in shared memory, joined in their order ------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < Q2; e++) {
            const int i = (n * 8 + 2 * t) / P + e;
            const float sum = sum_over_groups(l[n][e]);
            if (i < n_queries) {
                if (g == 0) {
                    sm_m[warp][i] = M[n][e];
                    sm_l[warp][i] = sum;
                }
#pragma unroll
                for (int j = 0; j < CH * 4; j++)
#pragma unroll
                    for (int r = 0; r < 2; r++)          // product j of a run of 64: dims 8 g + 2 j, + 1
                        sm_o[warp][i][(j >> 2) * 64 + 8 * g + 2 * (j & 3) + r] = P == 2 ? fmaf(o[j][n][2 * r + 1], 1.0f / SECOND, o[j][n][2 * r]) : o[j][n][2 * r + e];
            }
        }
    __syncthreads();
    // splits as a cluster: their results meet in the shared memory of its first block, behind that block's own warps' sums
    const size_t behind = sizeof(float) * WARPS * QT * (DMAX + 1);
    float* met = reinterpret_cast<float*>(smem + behind);             // [split][query][D + 2]
    if (a.in_cluster) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // the first block has left its stages
        met = cg::this_cluster().map_shared_rank(met, 0);
    }
    for (int idx = tid; idx < n_queries * D; idx += WARPS * 32) {
        const int i = idx / D, d = idx - i * D, qi = tile * QT + i;
        float m = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) m = fmaxf(m, sm_m[w][i]);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            // a warp without a key has no maximum and zeros; what is NaN has no maximum either, and counts
            const float f = sm_m[w][i] == -INFINITY ? 1.0f : ex2(sm_m[w][i] - m);
            L = fmaf(sm_l[w][i], f, L);
            O = fmaf(sm_o[w][i][d], f, O);
        }
        const int row = at.row0 + token_of(qi), h = head_of(qi);
        if (a.num_splits == 1) {
            finish<T>(a, O, L, m, row, h, d);
        } else {
            float* part = a.in_cluster ? met + (split * QT + i) * (D + 2)
                                       : a.scratch + (((size_t)row * a.n_heads + h) * a.num_splits + split) * (D + 2);
            part[d] = O;
            if (d == 0) {
                part[D] = m;
                part[D + 1] = L;
            }
        }
    }
    if (a.in_cluster) {
        cg::this_cluster().sync();
        if (split != 0) return;
        for (int idx = tid; idx < n_queries * D; idx += WARPS * 32) {
            const int i = idx / D, d = idx - i * D, qi = tile * QT + i;
            float m = -INFINITY, L = 0.0f, O = 0.0f;
            for (int k = 0; k < a.num_splits; k++) m = fmaxf(m, met[(k * QT + i) * (D + 2) + D]);
            for (int k = 0; k < a.num_splits; k++) {
                const float* part = met + (k * QT + i) * (D + 2);
                const float f = part[D] == -INFINITY ? 1.0f : ex2(part[D] - m);
                L = fmaf(part[D + 1], f, L);
                O = fmaf(part[d], f, O);
            }
            finish<T>(a, O, L, m, at.row0 + token_of(qi), head_of(qi), d);
        }
    }
}

// The splits' partial results of a (row, head), joined in a fixed order: one block each.  The splits' factors meet in shared memory;
// then every thread sums its dims (at heads of 64 two threads share one, every other split each), eight splits at a time on their way.
constexpr int MAX_SPLITS = 256;

template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Args a) {
    __shared__ float factor[MAX_SPLITS];
    __shared__ float scratch[32];
    __shared__ float other[128];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, D = a.head_dim, h = blockIdx.x % a.n_heads, nth = blockIdx.x / a.n_heads;
    const Portion at = portion_of(a, blockIdx.y);
    if (nth >= at.n) return;
    const int row = at.row0 + nth;
    const float* part = a.scratch + ((size_t)row * a.n_heads + h) * a.num_splits * (D + 2);
    float m = -INFINITY, L = 0.0f;
    for (int s = tid; s < a.num_splits; s += 128) m = fmaxf(m, part[(size_t)s * (D + 2) + D]);
    m = block_max(m, scratch);
    for (int s = tid; s < a.num_splits; s += 128) {
        const float ms = part[(size_t)s * (D + 2) + D];
        const float f = ms == -INFINITY ? 1.0f : ex2(ms - m);       // no key: zeros; NaN: no maximum, and it counts
        factor[s] = f;
        L = fmaf(part[(size_t)s * (D + 2) + D + 1], f, L);
    }
    L = block_sum(L, scratch);                                       // factor is there for all after it
    const int shares = D <= 64 ? 2 : 1, width = 128 / shares, share = tid / width;
    for (int d0 = 0; d0 < D; d0 += width) {
        const int d = d0 + tid % width;
        float O = 0.0f;
        if (d < D) {
#pragma unroll 8
            for (int s = share; s < a.num_splits; s += shares) O = fmaf(part[(size_t)s * (D + 2) + d], factor[s], O);
        }
        if (shares == 2) {
            other[tid] = O;
            __syncthreads();
            if (share == 0) O += other[tid + width];
        }
        if (d < D && share == 0) finish<T>(a, O, L, m, row, h, d);
    }
}

constexpr int MAX_CLUSTER = 8;           // splits up to here join in a cluster, if the blocks are of single tokens' size

// A kernel with more shared memory than a launch has by itself; the kernel is told so once on each device.
template <auto KERNEL>
int start(const Args& a, dim3 grid, int threads, int smem, int most_smem, cudaStream_t stream) {
    static std::atomic<unsigned long long> told{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const unsigned long long bit = 1ull << (device & 63);
    if (!(told.load() & bit) || device > 63) {
        e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem);
        if (e != cudaSuccess) return (int)e;
        told.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (a.in_cluster) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = a.num_splits;
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
    e = cudaLaunchKernelEx(&cfg, KERNEL, a);
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// Whether the queries of a (request, key/value head) are more columns than one tile has.
inline bool is_wide(long long queries, int head_dim, int dtype) { return queries * (dtype == SANDY_F32 ? 2 : 1) > 8 && head_dim <= 128; }

template <typename T, int CODE>
int launch(const Args& a, int n_z, int max_queries, int max_n, cudaStream_t stream) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;
    const bool wide = is_wide(max_queries, a.head_dim, sizeof(T) == 4 ? SANDY_F32 : SANDY_BF16);
    const bool one = P == 1 && max_queries == 1;
    int e;
#define LAUNCH(WARPS, DMAX, DK, NT, KT, RUN, ...)                                                                                \
    do {                                                                                                                         \
        constexpr int QT = 8 * NT / P, ring = WARPS * STAGES * 2 * KT * 16 * DMAX, sums = WARPS * QT * (DMAX + 1) * 4; \
        constexpr int alone = std::max(ring, sums), together = std::max(ring, sums + MAX_CLUSTER * QT * (DMAX + 2) * 4);          \
        e = start<attention_8bit_kernel<T, CODE, WARPS, DMAX, DK, NT, KT, RUN __VA_OPT__(,) __VA_ARGS__>>(                                                 \
            a, dim3((unsigned)((max_queries + QT - 1) / QT * a.num_splits), a.n_kv_heads, n_z), WARPS * 32,                      \
            a.in_cluster ? together : alone, NT == 1 ? together : alone, stream);                                                \
    } while (0)
    if (a.page_size % 8 != 0) {                          // rows one by one
        if (a.head_dim <= 64) LAUNCH(4, 64, 0, 1, 1, 0);
        else if (a.head_dim <= 128) LAUNCH(4, 128, 0, 1, 1, 0);
        else LAUNCH(4, 256, 0, 1, 1, 0);
    } else if (a.page_size % 16 == 0 && a.head_dim == 64) {
        if (wide) LAUNCH(4, 64, 64, 4, 1, 16);
        else if (a.two_warps && one) LAUNCH(2, 64, 64, 1, 2, 16, P == 1);
        else if (a.two_warps) LAUNCH(2, 64, 64, 1, 2, 16);
        else if (one) LAUNCH(4, 64, 64, 1, 2, 16, P == 1);
        else LAUNCH(4, 64, 64, 1, 2, 16);
    } else if (a.page_size % 16 == 0 && a.head_dim == 128) {
        if (wide) LAUNCH(4, 128, 128, 2, 1, 16);
        else if (one) LAUNCH(4, 128, 128, 1, 1, 16, P == 1);
        else LAUNCH(4, 128, 128, 1, 1, 16);
    } else if (a.head_dim <= 64) {
        if (wide) LAUNCH(4, 64, 0, 4, 1, 8);
        else LAUNCH(4, 64, 0, 1, 2, 8);
    } else if (a.head_dim <= 128) {
        if (wide) LAUNCH(4, 128, 0, 2, 1, 8);
        else LAUNCH(4, 128, 0, 1, 1, 8);
    } else {
        LAUNCH(4, 256, 0, 1, 1, 8);
    }
#undef LAUNCH
    if (e != SANDY_OK || a.num_splits == 1 || a.in_cluster) return e;
    return sandy_launch(join_kernel<T>, dim3((unsigned)((long long)max_n * a.n_heads), n_z), dim3(128), 0, stream, a);
}

}  // namespace

// How many blocks share a request's keys (max_keys: the most that one of its queries may see): as many as fill the SMs once (four
// blocks of single tokens an SM, two of a portion's), none with fewer than 128 keys, and no cluster of 6 or 7 (they fit an SM group
// badly); *scratch_floats: what their partial results take.
SANDY_API int sandy_attention_8bit_splits(int n_rows, int n_z, int max_n, int n_heads, int n_kv_heads, int head_dim, int max_keys,
                                          int dtype, int asked, long long* scratch_floats) {
    if (n_z < 1 || max_n < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || max_keys < 1 || asked < 0) return 1;
    const long long queries = (long long)max_n * (n_heads / n_kv_heads);
    const bool wide = is_wide(queries, head_dim, dtype);
    long long splits = asked;
    if (!asked) {
        const long long columns = queries * (dtype == SANDY_F32 ? 2 : 1), tile = !wide ? 8 : head_dim <= 64 ? 32 : 16;
        const long long blocks = (columns + tile - 1) / tile * n_kv_heads * n_z, room = (long long)sandy_sm_count() * (wide ? 2 : 4);
        splits = std::min(room / blocks, (long long)(max_keys + 127) / 128);
        if (!wide && (splits == 6 || splits == 7)) splits = 5;
        splits = std::max(1ll, std::min(splits, (long long)MAX_SPLITS));
    }
    if (scratch_floats) *scratch_floats = splits > (wide ? 1 : MAX_CLUSTER) ? (long long)n_rows * n_heads * splits * (head_dim + 2) : 0;
    return (int)splits;
}

// Attention of prompt portions or of single tokens (cache8.h).  max_keys: the most keys that one of a request's blocks of queries sees, by
// which the splits are cut; `scratch` as sandy_attention_8bit_splits says.  A row without a visible key becomes zeros.  Bit 4 of *status:
// a visible key without a page, a token of no request, or rows past n_rows.
SANDY_API int sandy_attention_8bit(const SandyAttend8* r, cudaStream_t stream) {
    if (!r) return SANDY_ERR_ARGUMENT;
    const SandyCache8& c = r->cache;
    const SandyAttentionRules& rules = r->rules;
    if (r->n_z == 0 || r->max_n == 0) return SANDY_OK;
    if (!r->q || !r->out || !r->positions || !(r->token_seq || r->q_start) || !c.k || !c.v || !c.k_scale || !c.v_scale || !c.block_table ||
        r->n_z < 0 || r->max_n < 0 || c.n_seqs < 1 || c.max_blocks < 1 || c.page_size < 1 || r->max_keys < 1 || r->num_splits < 1)
        return SANDY_ERR_ARGUMENT;
    if (rules.dist_bias && rules.n_dist < 1) return SANDY_ERR_ARGUMENT;
    if (rules.window < 0 || rules.keep_first < 0 || rules.chunk < 0 || !(rules.softcap >= 0.0f) || (rules.keep_first > 0 && rules.chunk > 0) ||
        (rules.elem_gate && rules.gate_dim < 1))
        return SANDY_ERR_UNSUPPORTED;
    if (c.head_dim < 16 || c.head_dim % 16 || c.head_dim > 256 || c.n_kv_heads < 1 || r->n_heads % c.n_kv_heads) return SANDY_ERR_UNSUPPORTED;
    if (c.page_stride % 16 || (((uintptr_t)c.k | (uintptr_t)c.v) & 15) || r->n_z > 65535 || c.n_kv_heads > 65535) return SANDY_ERR_UNSUPPORTED;
    const int group = r->n_heads / c.n_kv_heads, es = c.dtype == SANDY_F32 ? 4 : 2;
    const long long queries = (long long)r->max_n * group;
    if (queries > (1 << 28) || queries * r->num_splits > 0x7fffffffll || (long long)r->max_n * r->n_heads > 0x7fffffffll || r->num_splits > MAX_SPLITS)
        return SANDY_ERR_UNSUPPORTED;
    const bool in_cluster = r->num_splits > 1 && r->num_splits <= MAX_CLUSTER && !is_wide(queries, c.head_dim, c.dtype);
    if (r->num_splits > 1 && !in_cluster && !r->scratch) return SANDY_ERR_ARGUMENT;
    Args a = {};
    a.q = r->q;
    a.k = (const uint8_t*)c.k;
    a.v = (const uint8_t*)c.v;
    a.k_scale = c.k_scale;
    a.v_scale = c.v_scale;
    a.block_table = c.block_table;
    a.token_seq = r->token_seq;
    a.positions = r->positions;
    a.q_start = r->q_start;
    a.out = r->out;
    a.scratch = r->scratch;
    a.status = c.status;
    a.sink = rules.sink;
    a.out_gate = rules.out_gate;
    a.dist_bias = rules.dist_bias;
    a.elem_gate = rules.elem_gate;
    a.ld_q = r->ld_q;
    a.ld_out = r->ld_out;
    a.page_stride = c.page_stride;
    a.scale_stride = c.scale_stride;
    a.max_blocks = c.max_blocks;
    a.n_rows = r->n_rows;
    a.max_n = r->max_n;
    a.n_seqs = c.n_seqs;
    a.n_heads = r->n_heads;
    a.n_kv_heads = c.n_kv_heads;
    a.head_dim = c.head_dim;
    a.page_size = c.page_size;
    a.num_pages = c.num_pages;
    a.num_splits = r->num_splits;
    // a split's tiles of 16 keys, an even number; two more for the ends of a window and of the kept keys
    a.split_tiles = (((r->max_keys - 1) / 16 + 3 + r->num_splits - 1) / r->num_splits + 1) / 2 * 2;
    a.group = group;
    a.page_shift = (c.page_size & (c.page_size - 1)) == 0 ? __builtin_ctz(c.page_size) : -1;
    a.window = rules.window;
    a.keep_first = rules.keep_first;
    a.chunk = rules.chunk;
    a.n_dist = rules.n_dist;
    a.ld_elem_gate = rules.ld_elem_gate;
    a.gate_dim = rules.gate_dim;
    a.scale = r->scale;
    a.softcap = rules.softcap;
    a.in_cluster = in_cluster;
    // Blocks by the thousand, one for a (token, key/value head): what a block does before its keys and after them is paid once a warp, and
    // other blocks are there to hide the copies' latency.  256 tokens x 12 heads of 64 with 300 keys: 38 us in blocks of two warps,
    // 48 in blocks of four; 256 x 25 with 1,000 keys: 162 and 178.  Below four rounds of blocks the longest ones are left alone at the
    // end: 64 x 25 with 2,000 keys: 93 and 86; 32 x 12 with 1,000: 28 and 19.  Heads of 128 (256 x 8): 79 and 74.
    a.two_warps = r->num_splits == 1 && !r->q_start && (long long)r->n_z * c.n_kv_heads >= 16ll * sandy_sm_count();
    a.q_aligned = (((uintptr_t)r->q | (uintptr_t)(r->ld_q * es)) & 15) == 0;
    if (c.dtype == SANDY_F32 && c.code == SANDY_E4M3) return launch<float, SANDY_E4M3>(a, r->n_z, (int)queries, r->max_n, stream);
    if (c.dtype == SANDY_F32 && c.code == SANDY_INT8) return launch<float, SANDY_INT8>(a, r->n_z, (int)queries, r->max_n, stream);
    if (c.dtype == SANDY_BF16 && c.code == SANDY_E4M3) return launch<bf16, SANDY_E4M3>(a, r->n_z, (int)queries, r->max_n, stream);
    if (c.dtype == SANDY_BF16 && c.code == SANDY_INT8) return launch<bf16, SANDY_INT8>(a, r->n_z, (int)queries, r->max_n, stream);
    return SANDY_ERR_UNSUPPORTED;
}
