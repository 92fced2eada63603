// The paged key/value cache in 8 bits: a step's keys and values quantised as they are written, and cached rows read back.
//
// Formulas (blocks, codes and scales in kv_8bit.cuh).  A step's new tokens of a request touch pages kv_before / page_size to
// (kv_before + n - 1) / page_size of it.  For each touched block:
//   need = the scale for the largest |x| of the step's values in it;
//   s'   = need, if the block's first position is among the new ones; else max(s, need), and the codes c of the positions
//          before the step become round(c * s / s') where s' > s;
//   the new codes are round(x / s').
// A page that starts with the step's tokens is thus a fresh one, whatever it held before; slots behind the new tokens are left
// as they are.
//
// What bounds it.  2 (keys, values) x 2 bytes in and 1 byte out a value: a copy's work.  One warp owns one block and holds the
// block's new values in registers between the maximum and the rounding (up to 1,024 values; larger blocks are read twice,
// the second time from the caches), so each value crosses the memory bus once.
// Measured: 24 prompts of 400 to 930 tokens, bfloat16, 25 heads of 64, appended in 35.7 us, 66% of 6.57 TB/s: under ncu 62% of the issue
// slots are taken (14 instructions for 32 values, the indexes and conversions) and a third of the waiting is for memory, with the 25
// warps an SM that 64 registers allow; a step's 8 tokens in 2.4 us, of which the work is a hundredth.
// Reading: 24 requests of 300 to 4,000 rows of 8 heads of 128 in 67 us, 80%; one request's 700 rows in 5 us, a
// launch and the chain from the table to the scale to the codes.
#include "cache8.h"
#include "kv_8bit.cuh"

static_assert(sizeof(SandyCache8) == 96 && sizeof(SandyRows8) == 152, "the layout callers lay down");

namespace {

constexpr int WARPS = 8;
constexpr int HELD = 4;            // pieces of 8 values that a lane holds: 32 lanes x 4 x 8 = 1,024 values

struct Planes {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    long long page_stride, scale_stride;
};

// Eight values as they lie in memory; ALIGNED: they start on 16 bytes.
template <typename T>
struct Eight {
    uint4 raw[sizeof(T) / 2];
    template <bool ALIGNED>
    __device__ __forceinline__ void load(const T* __restrict__ p) {
        if (ALIGNED) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        } else if (sizeof(T) == 4) {
            const unsigned* w = reinterpret_cast<const unsigned*>(p);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
            raw[0] = make_uint4(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16, h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    // the bits of the largest |x| as a float: as unsigned numbers floats without their sign keep their order, infinities and NaN above
    __device__ __forceinline__ unsigned largest() const {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint4 r = raw[i];
            if (sizeof(T) == 4) {
                m = max(max(m, r.x & 0x7fffffffu), max(r.y & 0x7fffffffu, max(r.z & 0x7fffffffu, r.w & 0x7fffffffu)));
            } else {
                const unsigned h = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
                m = max(h << 16, h & 0xffff0000u);
            }
        }
        return m;
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const unsigned w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (sizeof(T) == 4) {
                    x[(4 * i + e) & 7] = __uint_as_float(w[e]);
                } else {
                    x[2 * e] = __uint_as_float(w[e] << 16);
                    x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                }
            }
        }
    }
};

// huge: some |x| of the block is above what a code times its scale may reach.
template <int CODE, typename T>
__device__ __forceinline__ uint2 encode8(const Eight<T>& values, float inv, bool huge) {
    float x[8];
    values.floats(x);
    if (huge) {
        const float most = __uint_as_float(LARGEST_KEPT_BITS);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = fminf(fmaxf(x[i], -most), most);
    }
    return make_uint2(encode4<CODE>(x[0], x[1], x[2], x[3], inv), encode4<CODE>(x[4], x[5], x[6], x[7], inv));
}

template <typename T, int CODE, bool ALIGNED>
__global__ void __launch_bounds__(WARPS * 32)
append_kernel(const T* __restrict__ k_src, const T* __restrict__ v_src, long long ld_k, long long ld_v, Planes cache,
              const int* __restrict__ block_table, int max_blocks, const int* __restrict__ q_start,
              const int* __restrict__ kv_before, int n_rows, int n_kv_heads, int head_dim, int page_size, int num_pages,
              int page_shift, int row_shift, int max_len, int* __restrict__ status) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.z, nth = blockIdx.x;                     // which of the request's touched pages
    const int unit = blockIdx.y * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int first_row = q_start[s], n = q_start[s + 1] - first_row, before = kv_before[s];
    if (unit >= 2 * n_kv_heads || n <= 0) return;
    // rows that are not there, or more than max_len said: then there may be no block for the last pages; positions that are no int
    if (first_row < 0 || n > n_rows - first_row || n > max_len || (long long)before + n + page_size > 0x7fffffffll) {
        if (lane == 0 && status) atomicOr(status, 8);
        return;
    }
    const int block = (page_shift >= 0 ? before >> page_shift : before / page_size) + nth;
    const int lo = max(before, block * page_size), hi = min(before + n, (block + 1) * page_size);     // new positions in the block
    if (lo >= hi && before >= 0) return;
    // the values, which hang on no page, and at the same time the page and the block's old scale
    const int h = unit >> 1, plane = unit & 1;                      // neighbouring warps: keys and values of one head
    const long long ld = plane ? ld_v : ld_k;
    const T* src = (plane ? v_src : k_src) + (size_t)(first_row + max(lo - before, 0)) * ld + (size_t)h * head_dim;
    const int per_row = head_dim >> 3, pieces = before >= 0 ? (hi - lo) * per_row : 0;
    Eight<T> x[HELD];
#pragma unroll
    for (int k = 0; k < HELD; k++) {
        const int i = lane + 32 * k, row = row_shift >= 0 ? i >> row_shift : i / per_row;
        if (i < pieces) x[k].template load<ALIGNED>(src + (size_t)row * ld + (i - row * per_row) * 8);
        else x[k].clear();
    }
    const int page = before >= 0 && block < max_blocks ? block_table[(size_t)s * max_blocks + block] : -1;
    if (page < 0 || page >= num_pages) {                            // no page behind these positions: nothing may be written
        if (lane == 0 && unit == 0 && status) atomicOr(status, 8);
        return;
    }
    uint8_t* codes = (plane ? cache.v : cache.k) + (size_t)page * cache.page_stride + (size_t)h * page_size * head_dim;
    float* scale_at = (plane ? cache.v_scale : cache.k_scale) + (size_t)page * cache.scale_stride + h;
    const int kept = lo - block * page_size;                        // positions of the block that were there before
    const float old = kept > 0 ? *scale_at : 0.0f;

    unsigned amax = 0;
#pragma unroll
    for (int k = 0; k < HELD; k++) amax = max(amax, x[k].largest());
    for (int i = lane + 32 * HELD; i < pieces; i += 32) {
        Eight<T> y;
        y.template load<ALIGNED>(src + (size_t)(i / per_row) * ld + (i % per_row) * 8);
        amax = max(amax, y.largest());
    }
    amax = __reduce_max_sync(0xffffffffu, amax);

    const float nan = __uint_as_float(0x7fffffffu);
    float now = amax >= 0x7f800000u ? nan : scale_for<CODE>(min(amax, LARGEST_KEPT_BITS));
    if (kept > 0 && !(old <= now)) now = old;                       // the old one is larger, or one of the two is NaN
    if (amax >= 0x7f800000u) now = nan;
    const bool sound = now == now, huge = amax > LARGEST_KEPT_BITS;
    const float inv = sound ? 1.0f / now : 0.0f;                    // of a power of two: exact

    if (kept > 0 && sound && now > old) {                           // the block's earlier codes at its new scale
        const float shrink = old * inv;
        for (int i = lane; i < kept * (head_dim >> 2); i += 32) {
            unsigned* w = reinterpret_cast<unsigned*>(codes) + i;
            unsigned a, b;
            decode4<CODE>(*w, a, b);
            const float2 p = half2_floats(a), q = half2_floats(b);
            *w = encode4<CODE>(p.x, p.y, q.x, q.y, shrink);
        }
    }
    uint2* dst = reinterpret_cast<uint2*>(codes + (size_t)kept * head_dim);      // the new rows follow one another in a block
#pragma unroll
    for (int k = 0; k < HELD; k++) {
        const int i = lane + 32 * k;
        if (i < pieces) dst[i] = sound ? encode8<CODE>(x[k], inv, huge) : make_uint2(0u, 0u);
    }
    for (int i = lane + 32 * HELD; i < pieces; i += 32) {
        Eight<T> y;
        y.template load<ALIGNED>(src + (size_t)(i / per_row) * ld + (i % per_row) * 8);
        dst[i] = sound ? encode8<CODE>(y, inv, huge) : make_uint2(0u, 0u);
    }
    if (lane == 0) *scale_at = now;
}

// Sixteen codes times their scale, rounded to T (exact in bfloat16 and float32 for the scales that appending gives).
template <typename T, int CODE>
__device__ __forceinline__ void store16(uint4 raw, float scale, T* dst, bool aligned) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned a, b;
        decode4<CODE>(w[i], a, b);
        const float2 p = half2_floats(a), q = half2_floats(b);
        x[4 * i] = p.x * scale; x[4 * i + 1] = p.y * scale; x[4 * i + 2] = q.x * scale; x[4 * i + 3] = q.y * scale;
    }
    if (aligned) {
        if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                reinterpret_cast<float4*>(dst)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
            __nv_bfloat162 h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<const uint4*>(h)[0];
            reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<const uint4*>(h)[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) dst[i] = from_f32<T>(x[i]);
    }
}

constexpr int READ_THREADS = 256;
constexpr int READ_ROWS = 8;       // rows of a request that a block reads

// A lane takes 16 codes of the keys and as many of the values; neighbouring lanes follow the output row, which is written
// whole lines at a time.
template <typename T, int CODE>
__global__ void __launch_bounds__(READ_THREADS)
read_kernel(Planes cache, const int* __restrict__ block_table, int max_blocks, const int* __restrict__ first,
            const int* __restrict__ out_start, T* __restrict__ k_out, T* __restrict__ v_out, long long ld_k, long long ld_v,
            int n_rows, int max_len, int n_kv_heads, int head_dim, int page_size, int num_pages, bool aligned, int* __restrict__ status) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.y;
    const int row0 = out_start[s], n = out_start[s + 1] - row0, from = first[s];
    const int r0 = blockIdx.x * READ_ROWS, rows = min(READ_ROWS, n - r0);
    if (rows <= 0) return;
    if (row0 < 0 || n > n_rows - row0 || n > max_len) {             // rows that are not there, or more than max_len said
        if (threadIdx.x == 0 && status) atomicOr(status, 16);
        return;
    }
    const int per_head = head_dim >> 4, per_row = n_kv_heads * per_head;
    for (int i = threadIdx.x; i < rows * per_row; i += READ_THREADS) {
        const int r = i / per_row, at = i % per_row, h = at / per_head, d = at % per_head * 16;
        const int pos = from + r0 + r;
        const int block = pos >= 0 ? pos / page_size : max_blocks;
        const int page = block < max_blocks ? block_table[(size_t)s * max_blocks + block] : -1;
        if (page < 0 || page >= num_pages) {                        // no page behind this position: its row is left as it was
            if (at == 0 && status) atomicOr(status, 16);
            continue;
        }
        const size_t code_at = (size_t)page * cache.page_stride + ((size_t)h * page_size + (pos - block * page_size)) * head_dim + d;
        const size_t scale_at = (size_t)page * cache.scale_stride + h;
        const uint4 kc = *reinterpret_cast<const uint4*>(cache.k + code_at);
        const uint4 vc = *reinterpret_cast<const uint4*>(cache.v + code_at);
        const float ks = cache.k_scale[scale_at], vs = cache.v_scale[scale_at];
        store16<T, CODE>(kc, ks, k_out + (size_t)(row0 + r0 + r) * ld_k + (size_t)h * head_dim + d, aligned);
        store16<T, CODE>(vc, vs, v_out + (size_t)(row0 + r0 + r) * ld_v + (size_t)h * head_dim + d, aligned);
    }
}

// Sizes both entries refuse.
int refused(const SandyRows8* r) {
    const SandyCache8& c = r->cache;
    if (!r->k_rows || !r->v_rows || !r->start || !r->first || !c.k || !c.v || !c.k_scale || !c.v_scale || !c.block_table || c.n_seqs < 0 ||
        r->max_len < 0 || c.n_kv_heads < 1 || c.head_dim < 16 || c.page_size < 1 || c.page_stride < 1)
        return SANDY_ERR_ARGUMENT;
    if (c.head_dim % 16 || c.page_stride % 16 || (((uintptr_t)c.k | (uintptr_t)c.v) & 15) || c.n_seqs > 65535) return SANDY_ERR_UNSUPPORTED;
    return SANDY_OK;
}

template <typename T>
bool on_16_bytes(const SandyRows8& r) {
    return (((uintptr_t)r.k_rows | (uintptr_t)r.v_rows | (size_t)(r.ld_k * (long long)sizeof(T)) | (size_t)(r.ld_v * (long long)sizeof(T))) & 15) == 0;
}

}  // namespace

// Quantises rows (cache8.h) into their pages.  Pages that two requests of one call both write are not allowed.  Bit 3 of *status: a
// position without a page, or rows past n_rows.
SANDY_API int sandy_kv_append_8bit(const SandyRows8* r, cudaStream_t stream) {
    if (!r) return SANDY_ERR_ARGUMENT;
    const SandyCache8& c = r->cache;
    if (c.n_seqs == 0 || r->max_len == 0) return SANDY_OK;
    if (const int code = refused(r)) return code;
    const int groups = (2 * c.n_kv_heads + WARPS - 1) / WARPS;
    const long long touched = ((long long)r->max_len + c.page_size - 2) / c.page_size + 1;      // by one request, wherever it starts
    if (touched > 0x7fffffffll || groups > 65535) return SANDY_ERR_UNSUPPORTED;
    const Planes cache = {(uint8_t*)c.k, (uint8_t*)c.v, c.k_scale, c.v_scale, c.page_stride, c.scale_stride};
    const dim3 grid((unsigned)touched, groups, c.n_seqs), block(WARPS * 32);
    auto shift = [](int n) { return (n & (n - 1)) == 0 ? __builtin_ctz(n) : -1; };      // -1: no power of two
#define APPEND(T, CODE)                                                                                                         \
    return sandy_launch(on_16_bytes<T>(*r) ? append_kernel<T, CODE, true> : append_kernel<T, CODE, false>, grid, block, 0, stream, \
                        (const T*)r->k_rows, (const T*)r->v_rows, r->ld_k, r->ld_v, cache, c.block_table, c.max_blocks, r->start, \
                        r->first, r->n_rows, c.n_kv_heads, c.head_dim, c.page_size, c.num_pages, shift(c.page_size), \
                        shift(c.head_dim / 8), r->max_len, c.status)
    if (c.dtype == SANDY_F32 && c.code == SANDY_E4M3) APPEND(float, SANDY_E4M3);
    if (c.dtype == SANDY_F32 && c.code == SANDY_INT8) APPEND(float, SANDY_INT8);
    if (c.dtype == SANDY_BF16 && c.code == SANDY_E4M3) APPEND(bf16, SANDY_E4M3);
    if (c.dtype == SANDY_BF16 && c.code == SANDY_INT8) APPEND(bf16, SANDY_INT8);
#undef APPEND
    return SANDY_ERR_UNSUPPORTED;
}

// The rows become the cached numbers.  Bit 4 of *status: a position without a page, or rows past n_rows.
SANDY_API int sandy_kv_read_8bit(const SandyRows8* r, cudaStream_t stream) {
    if (!r) return SANDY_ERR_ARGUMENT;
    const SandyCache8& c = r->cache;
    if (c.n_seqs == 0 || r->max_len == 0) return SANDY_OK;
    if (const int code = refused(r)) return code;
    const Planes cache = {(uint8_t*)c.k, (uint8_t*)c.v, c.k_scale, c.v_scale, c.page_stride, c.scale_stride};
    const dim3 grid((r->max_len - 1) / READ_ROWS + 1, c.n_seqs), block(READ_THREADS);
#define READ(T, CODE)                                                                                                           \
    return sandy_launch(read_kernel<T, CODE>, grid, block, 0, stream, cache, c.block_table, c.max_blocks, r->first, r->start,    \
                        (T*)r->k_rows, (T*)r->v_rows, r->ld_k, r->ld_v, r->n_rows, r->max_len, c.n_kv_heads, c.head_dim, c.page_size, \
                        c.num_pages, on_16_bytes<T>(*r), c.status)
    if (c.dtype == SANDY_F32 && c.code == SANDY_E4M3) READ(float, SANDY_E4M3);
    if (c.dtype == SANDY_F32 && c.code == SANDY_INT8) READ(float, SANDY_INT8);
    if (c.dtype == SANDY_BF16 && c.code == SANDY_E4M3) READ(bf16, SANDY_E4M3);
    if (c.dtype == SANDY_BF16 && c.code == SANDY_INT8) READ(bf16, SANDY_INT8);
#undef READ
    return SANDY_ERR_UNSUPPORTED;
}
