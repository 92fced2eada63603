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
// consecutive dims of keys 2t, 2t+1, 2t+8, 2t+9 (t = lane % 4), whose bytes are paired by a byte permutation.  So codes go from
// memory to registers to the tensor cores, with no shared memory and no barrier between them.  S comes out with keys in the lane
// groups; movmatrix turns P, as half-precision pairs, into the operand of the second product.
//
// Scales.  A score is S * sk * (2^eq * scale), a factor a key.  A value's scale joins the weight: with M the running maximum of
// s_j + log2(sv_j) (s in units of log 2), p_j = 2^(s_j - M) is summed for the denominator and p_j * sv_j <= 1 (2 if the scale is
// no power of two) is rounded to half precision for the product.  No block's values are out of half precision's range
// this way, and nothing is lost that would count beside the largest term.
//
// Roundings.  q is scaled by a power of two (2^eq) so that its largest element lies in [1, 2) and rounded to half precision:
// exact for bfloat16 elements above 2^-14 of the largest, off by 2^-25 of it at most.  P rounds to 11 bits, the row sum is taken
// before.  For float32 both are split into two half-precision pieces (22 bits), which lie in neighbouring columns; the two
// columns' results are in the same lane and are added there.
//
// What bounds it.  Single tokens: the codes' bytes.  A warp asks for 64 keys' codes at a time (4 KB of keys and 4 KB of values
// at heads of 64), so 16 warps an SM keep more than 100 KB on their way; a block's four warps take turns along the keys, and
// `num_splits` blocks share a request's keys where there are few requests (partial results in scratch, joined by a second
// kernel in a fixed order).  Prompt portions: the tensor cores' warp-level instructions.
#include "attention_rules.h"
#include "kv_8bit.cuh"

namespace {

constexpr int WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f;

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
    int max_blocks, n_rows, n_seqs, n_heads, n_kv_heads, head_dim, page_size, num_pages, num_splits;
    int window, keep_first, chunk, n_dist, ld_elem_gate, gate_dim;
    float scale, softcap;
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
    if (p.row0 < 0 || p.n > a.n_rows - p.row0) {                     // rows that are not there
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

// DMAX: 64, 128 or 256, the head size rounded up; NT: column tiles of 8; KT: key tiles of 16 that a warp takes at a time.
template <typename T, int CODE, int DMAX, int NT, int KT>
__global__ void __launch_bounds__(WARPS * 32)
attention_8bit_kernel(const __grid_constant__ Args a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;            // pieces a number is split into
    constexpr int QT = 8 * NT / P;                       // queries of a block
    constexpr int CH = DMAX / 64;                        // runs of 64 dims
    constexpr int Q2 = 2 / P;                            // queries in a lane's two columns of a tile
    __shared__ float sm_o[WARPS][QT][DMAX + 1];
    __shared__ float sm_m[WARPS][QT], sm_l[WARPS][QT];

    pdl_launch_dependents();
    pdl_wait();
    const int z = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x % a.num_splits, tile = blockIdx.x / a.num_splits;
    const Portion at = portion_of(a, z);
    const int group = a.n_heads / a.n_kv_heads;
    const int n_queries = min(QT, at.n * group - tile * QT);         // of this block
    if (n_queries <= 0) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int D = a.head_dim, ps = a.page_size;

    // ---- q: column g of every tile, as the second operand ------------------------------------------------------
    unsigned qf[NT][CH * 4][2];
    float my_factor[NT];                                 // of column g
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int i = (n * 8 + g) / P, qi = tile * QT + i;
        const bool there = i < n_queries;
        const T* src = (const T*)a.q + (size_t)(at.row0 + (there ? qi / group : 0)) * a.ld_q + (size_t)(kvh * group + (there ? qi % group : 0)) * D;
        unsigned amax = 0;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int d = 64 * c + 16 * t + e;
                if (there && 64 * c + 16 * t < D) amax = max(amax, __float_as_uint(to_f32(src[d])) & 0x7fffffffu);
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
                float x0 = 0.0f, x1 = 0.0f;
                if (there && 64 * c + 16 * t < D) {
                    x0 = to_f32(src[64 * c + 16 * t + 2 * w]) * down;
                    x1 = to_f32(src[64 * c + 16 * t + 2 * w + 1]) * down;
                }
                if (P == 2 && (g & 1)) {                 // the second piece: what the first one leaves
                    x0 -= __half2float(__float2half_rn(x0));
                    x1 -= __half2float(__float2half_rn(x1));
                }
                qf[n][c * 4 + (w >> 1)][w & 1] = pack_half(x0, x1);
            }
    }
    // the lane's two columns 2t, 2t + 1 of every tile: one query each, or the two pieces of one
    float factor[NT][Q2];
    int pos[NT][Q2], lo[NT][Q2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < Q2; e++) {
            const int i = (n * 8 + 2 * t) / P + e;
            factor[n][e] = __shfl_sync(0xffffffffu, my_factor[n], (2 * t + e) * 4);
            pos[n][e] = i < n_queries ? at.before + (tile * QT + i) / group : -1;
            lo[n][e] = first_key(a, max(pos[n][e], 0));
        }

    // ---- the block's keys, as tiles of 16 positions: kept first ones, then from the first query's first to the last query's own ----
    const int pos_first = at.before + tile * QT / group, pos_last = at.before + (tile * QT + n_queries - 1) / group;
    const int lo_first = first_key(a, max(pos_first, 0));
    const int kept_tiles = lo_first > 0 ? min((a.keep_first + 15) >> 4, lo_first >> 4) : 0;
    const bool known = (unsigned)at.seq < (unsigned)a.n_seqs;
    if (!known && tid == 0 && a.status) atomicOr(a.status, 16);
    const int n_tiles = known && pos_last >= 0 ? kept_tiles + (pos_last >> 4) - (lo_first >> 4) + 1 : 0;
    const int per_split = ((n_tiles + a.num_splits - 1) / a.num_splits + KT - 1) / KT * KT;
    const int tile_end = min(n_tiles, (split + 1) * per_split);
    const int* table = a.block_table + (size_t)(known ? at.seq : 0) * a.max_blocks;
    const bool whole_pages = (ps & 15) == 0;             // a tile of 16 keys lies in one page

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
    const size_t head_at = (size_t)kvh * ps * D;

    for (int it = split * per_split + warp * KT; it < tile_end; it += WARPS * KT) {
        uint4 kw[KT][2][CH];                              // keys g, g + 8: dims 64 c + 16 t ..
        uint2 vw[KT][4][CH];                              // keys 2t, 2t + 1, 2t + 8, 2t + 9: dims 64 c + 8 g ..
        float ks[KT][2], vs[KT][2];                       // scales of keys g, g + 8
        int key0[KT];                                     // the tile's first position
        unsigned there = 0;                               // bit 2 kt + r: key g + 8 r of tile kt has a page
        // A tile's loads: which key, its page, then codes and scales.  Rows that no query of the block sees are zeros.
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            const int nth = it + kt;
            key0[kt] = (nth < kept_tiles ? nth : nth - kept_tiles + (lo_first >> 4)) << 4;
            const bool in = nth < tile_end;
            auto seen = [&](int j) { return in && j <= pos_last && (j >= lo_first || j < a.keep_first); };
            int tile_page = -1, slot0 = 0;
            if (whole_pages && in) {
                const int b = key0[kt] / ps;
                slot0 = key0[kt] - b * ps;
                tile_page = b < a.max_blocks ? table[b] : -1;
            }
            auto row_of = [&](int j, size_t& off, int& page) {       // false: no such row
                int slot = slot0 + (j - key0[kt]);
                page = tile_page;
                if (!seen(j)) return false;
                if (!whole_pages) {
                    const int b = j / ps;
                    slot = j - b * ps;
                    page = b < a.max_blocks ? table[b] : -1;
                }
                if (page < 0 || page >= a.num_pages) {
                    if (a.status) atomicOr(a.status, 16);
                    return false;
                }
                off = (size_t)page * a.page_stride + head_at + (size_t)slot * D;
                return true;
            };
#pragma unroll
            for (int r = 0; r < 2; r++) {
                size_t off = 0;
                int page = 0;
                const bool ok = row_of(key0[kt] + g + 8 * r, off, page);
                if (ok) there |= 1u << (2 * kt + r);
                ks[kt][r] = ok ? a.k_scale[(size_t)page * a.scale_stride + kvh] : 0.0f;
                vs[kt][r] = ok ? a.v_scale[(size_t)page * a.scale_stride + kvh] : 0.0f;
#pragma unroll
                for (int c = 0; c < CH; c++)
                    kw[kt][r][c] = ok && 64 * c + 16 * t < D ? __ldg(reinterpret_cast<const uint4*>(a.k + off + 64 * c + 16 * t))
                                                            : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                size_t off = 0;
                int page = 0;
                const bool ok = row_of(key0[kt] + 2 * t + (r & 1) + 8 * (r >> 1), off, page);
#pragma unroll
                for (int c = 0; c < CH; c++)
                    vw[kt][r][c] = ok && 64 * c + 8 * g < D ? __ldg(reinterpret_cast<const uint2*>(a.v + off + 64 * c + 8 * g)) : make_uint2(0u, 0u);
            }
        }

        // ---- S, and the scores in units of log 2 -----------------------------------------------------------------
        float sc[KT][NT][4];
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[kt][n][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const unsigned w0[4] = {kw[kt][0][c].x, kw[kt][0][c].y, kw[kt][0][c].z, kw[kt][0][c].w};
                const unsigned w1[4] = {kw[kt][1][c].x, kw[kt][1][c].y, kw[kt][1][c].z, kw[kt][1][c].w};
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
        float x[KT][NT][2][Q2], top[NT][Q2];              // [tile][column tile][key g, g + 8][query]
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < Q2; e++) top[n][e] = M[n][e];
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int j = key0[kt] + g + 8 * r;
                const bool ok = (there >> (2 * kt + r)) & 1;
                // log2 of the value's scale; of one that is not finite 0, so that its weight is NaN and the others stay numbers
                const int exponent = (int)(__float_as_uint(vs[kt][r]) >> 23) & 255;
                const float ev = exponent == 255 ? 0.0f : (float)(exponent - 127);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < Q2; e++) {
                        float s = (P == 2 ? sc[kt][n][2 * r] + sc[kt][n][2 * r + 1] : sc[kt][n][2 * r + e]) * (ks[kt][r] * factor[n][e]);
                        if (a.softcap > 0.0f) s = a.softcap * (P == 2 ? tanhf(s / a.softcap) : tanh_fast(s / a.softcap));
                        const bool visible = ok && j <= pos[n][e] && (j >= lo[n][e] || j < a.keep_first);
                        if (a.dist_bias && visible) {
                            const int h = kvh * group + (tile * QT + (n * 8 + 2 * t) / P + e) % group;
                            s += a.dist_bias[(size_t)h * a.n_dist + min(pos[n][e] - j, a.n_dist - 1)];
                        }
                        s = visible ? s * LOG2E : -INFINITY;
                        x[kt][n][r][e] = s;
                        top[n][e] = fmaxf(top[n][e], s + ev);
                    }
            }
        // ---- the running maximum; weights; P as the second operand ---------------------------------------------
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < Q2; e++) {
                const float m = max_over_groups(top[n][e]);
                const float shrink = m == -INFINITY ? 1.0f : ex2(M[n][e] - m);
                M[n][e] = m;
                l[n][e] *= shrink;
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
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            unsigned pf[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < Q2; e++) {
                        const float s = x[kt][n][r][e];
                        const bool none = s == -INFINITY;                        // not visible, or a score that weighs nothing
                        const float p = none ? 0.0f : ex2(s - M[n][e]);
                        l[n][e] += p;
                        w[e] = none ? 0.0f : p * vs[kt][r];
                    }
                    if (P == 2) w[1] = w[0] - __half2float(__float2half_rn(w[0]));
                    pf[n][r] = turn(pack_half(w[0], w[1]));
                }
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    unsigned w[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) w[r] = half ? vw[kt][r][c].y : vw[kt][r][c].x;
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

    // ---- the warps' states in shared memory, joined in their order ------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < Q2; e++) {
            const int i = (n * 8 + 2 * t) / P + e;
            const float sum = sum_over_groups(l[n][e]);
            if (g == 0) {
                sm_m[warp][i] = M[n][e];
                sm_l[warp][i] = sum;
            }
#pragma unroll
            for (int j = 0; j < CH * 4; j++)
#pragma unroll
                for (int r = 0; r < 2; r++)              // product j of a run of 64: dims 8 g + 2 j, + 1
                    sm_o[warp][i][(j >> 2) * 64 + 8 * g + 2 * (j & 3) + r] = P == 2 ? o[j][n][2 * r] + o[j][n][2 * r + 1] : o[j][n][2 * r + e];
        }
    __syncthreads();
    for (int idx = tid; idx < n_queries * D; idx += WARPS * 32) {
        const int i = idx / D, d = idx % D, qi = tile * QT + i;
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
        if (a.num_splits == 1) {
            finish<T>(a, O, L, m, at.row0 + qi / group, kvh * group + qi % group, d);
        } else {
            const size_t row = ((size_t)(at.row0 + qi / group) * a.n_heads + kvh * group + qi % group) * a.num_splits + split;
            float* part = a.scratch + row * (D + 2);
            part[d] = O;
            if (d == 0) {
                part[D] = m;
                part[D + 1] = L;
            }
        }
    }
}

// The splits' partial results of a (row, head), joined in their order: one warp each.
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Args a, int n_z) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const Portion at = portion_of(a, blockIdx.y);
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (unit >= at.n * a.n_heads) return;
    const int row = at.row0 + unit / a.n_heads, h = unit % a.n_heads, D = a.head_dim;
    const float* part = a.scratch + ((size_t)row * a.n_heads + h) * a.num_splits * (D + 2);
    float m = -INFINITY;
    for (int s = lane; s < a.num_splits; s += 32) m = fmaxf(m, part[(size_t)s * (D + 2) + D]);
    m = warp_max(m);
    for (int d = lane; d < D; d += 32) {
        float L = 0.0f, O = 0.0f;
        for (int s = 0; s < a.num_splits; s++) {
            const float* p = part + (size_t)s * (D + 2);
            const float f = p[D] == -INFINITY ? 1.0f : ex2(p[D] - m);
            L = fmaf(p[D + 1], f, L);
            O = fmaf(p[d], f, O);
        }
        finish<T>(a, O, L, m, row, h, d);
    }
}

template <typename T, int CODE>
int launch(const Args& a, int n_z, int max_queries, int max_n, cudaStream_t stream) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;
    const bool wide = max_queries * P > 8;               // more columns than one tile has
    int e;
#define RUN(DMAX, NT, KT)                                                                                                        \
    e = sandy_launch(attention_8bit_kernel<T, CODE, DMAX, NT, KT>,                                                               \
                     dim3((unsigned)((max_queries + 8 * NT / P - 1) / (8 * NT / P) * a.num_splits), a.n_kv_heads, n_z), dim3(WARPS * 32), 0, \
                     stream, a)
    if (a.head_dim <= 64) {
        if (wide) RUN(64, 4, 2);
        else RUN(64, 1, 4);
    } else if (a.head_dim <= 128) {
        if (wide) RUN(128, 2, 1);
        else RUN(128, 1, 2);
    } else {
        RUN(256, 1, 1);
    }
#undef RUN
    if (e != SANDY_OK || a.num_splits == 1) return e;
    return sandy_launch(join_kernel<T>, dim3((unsigned)(((long long)max_n * a.n_heads + 3) / 4), n_z), dim3(128), 0, stream, a, n_z);
}

}  // namespace

// How many blocks share a request's keys: as many as give every SM some four blocks, none with fewer than 16 keys x 16.
SANDY_API int sandy_attention_8bit_splits(int n_z, int max_n, int n_heads, int n_kv_heads, int head_dim, int max_keys, int dtype) {
    if (n_z < 1 || max_n < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || max_keys < 1) return 1;
    const long long queries = (long long)max_n * (n_heads / n_kv_heads), columns = queries * (dtype == SANDY_F32 ? 2 : 1);
    const long long tile = columns <= 8 || head_dim > 128 ? 8 : head_dim <= 64 ? 32 : 16;
    const long long blocks = (columns + tile - 1) / tile * n_kv_heads * n_z;
    const long long wanted = ((long long)sandy_sm_count() * 4 + blocks - 1) / blocks, most = (max_keys + 255) / 256;
    long long splits = wanted < most ? wanted : most;
    return (int)(splits < 1 ? 1 : splits > 256 ? 256 : splits);
}

// Attention of prompt portions (q_start [n_z + 1], positions = kv_before [n_z], token_seq null, request z = row z of the block
// table; max_n: the most tokens of one) or of single tokens (q_start null: token z of request token_seq[z] at positions[z]; max_n 1).
// q: [n_rows, H * D], out likewise, row pitches ld_q and ld_out (elements); k, v, scales and table as sandy_kv_append_8bit has them,
// n_seqs rows in the table.  num_splits > 1 needs `scratch`: n_rows * H * num_splits * (D + 2) floats.  A row without a visible key
// becomes zeros.  Bit 4 of *status: a visible key without a page, a token of no request, or rows past n_rows.
SANDY_API int sandy_attention_8bit(const void* q, long long ld_q, const void* k, const void* v, const float* k_scale,
                                   const float* v_scale, long long page_stride, long long scale_stride, const int* block_table,
                                   int max_blocks, int n_seqs, const int* token_seq, const int* positions, const int* q_start, void* out,
                                   long long ld_out, int n_rows, int n_z, int max_n, int n_heads, int n_kv_heads, int head_dim,
                                   int page_size, int num_pages, float scale, const SandyAttentionRules* rules, int num_splits, float* scratch,
                                   int dtype, int code, int* status, cudaStream_t stream) {
    if (n_z == 0 || max_n == 0) return SANDY_OK;
    if (!rules || !q || !k || !v || !k_scale || !v_scale || !block_table || !positions || !out || !(token_seq || q_start) || n_z < 0 ||
        max_n < 0 || n_seqs < 1 || max_blocks < 1 || page_size < 1 || num_splits < 1 || (num_splits > 1 && !scratch))
        return SANDY_ERR_ARGUMENT;
    if (rules->dist_bias && rules->n_dist < 1) return SANDY_ERR_ARGUMENT;
    if (rules->window < 0 || rules->keep_first < 0 || rules->chunk < 0 || !(rules->softcap >= 0.0f) ||
        (rules->keep_first > 0 && rules->chunk > 0) || (rules->elem_gate && rules->gate_dim < 1))
        return SANDY_ERR_UNSUPPORTED;
    if (head_dim < 16 || head_dim % 16 || head_dim > 256 || n_kv_heads < 1 || n_heads % n_kv_heads) return SANDY_ERR_UNSUPPORTED;
    if (page_stride % 16 || (((uintptr_t)k | (uintptr_t)v) & 15) || n_z > 65535 || n_kv_heads > 65535) return SANDY_ERR_UNSUPPORTED;
    const long long queries = (long long)max_n * (n_heads / n_kv_heads);
    if (queries > (1 << 28) || queries * num_splits > 0x7fffffffll) return SANDY_ERR_UNSUPPORTED;
    const Args a = {q, (const uint8_t*)k, (const uint8_t*)v, k_scale, v_scale, block_table, token_seq, positions, q_start, out, scratch,
                    status, rules->sink, rules->out_gate, rules->dist_bias, rules->elem_gate, ld_q, ld_out, page_stride, scale_stride,
                    max_blocks, n_rows, n_seqs, n_heads, n_kv_heads, head_dim, page_size, num_pages, num_splits, rules->window,
                    rules->keep_first, rules->chunk, rules->n_dist, rules->ld_elem_gate, rules->gate_dim, scale, rules->softcap};
    if (dtype == SANDY_F32 && code == SANDY_E4M3) return launch<float, SANDY_E4M3>(a, n_z, (int)queries, max_n, stream);
    if (dtype == SANDY_F32 && code == SANDY_INT8) return launch<float, SANDY_INT8>(a, n_z, (int)queries, max_n, stream);
    if (dtype == SANDY_BF16 && code == SANDY_E4M3) return launch<bf16, SANDY_E4M3>(a, n_z, (int)queries, max_n, stream);
    if (dtype == SANDY_BF16 && code == SANDY_INT8) return launch<bf16, SANDY_INT8>(a, n_z, (int)queries, max_n, stream);
    return SANDY_ERR_UNSUPPORTED;
}
