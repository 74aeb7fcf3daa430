// Attention of one new token per sequence over a paged cache (yuuka_attention_decode): the kernel.
//
// Mathematics. A unit is one KV head of one row of the batch, with up to 8 NT of the query heads that share it as columns.
// Its keys are taken 16 at a time: S^T = K Q^T (keys as the rows of the product, heads as its 8-wide columns), running
// maximum m and sum l per head, O^T += V^T P^T. Scores live in the base-2 domain, s = (scale log2 e) q.k, and probabilities
// carry a factor of 2^14, p = 2^(s - m + 14), so that those down to 2^-28 of the largest stay normal in f16.
//
// What bounds it: the bytes of the cache, read once. The products run on mma.sync: at 148 x 23 bytes a clock (the measured
// memory rate) they take 10 to 40 % of its issue rate, and operands go straight from the cache's own layout into fragments.
// The dimension that a product sums over may be taken in any order and a fragment's rows may stand for any dimensions, so a
// lane copies (cp.async) the 16 bytes of a key that it will itself multiply, and of V the same dimensions of four keys, whose
// halves one byte permutation pairs up: no lane reads what another has copied, no barrier, no bank conflict. (Q8_0's blocks of
// 34 bytes are copied by words, and the word at which a lane starts is chosen so that its two words are never misaligned.)
//
// Work is cut at the granularity of warps: all tiles of 16 keys of all units form one sequence, every warp of the grid takes
// an equal run of it, wherever that begins and ends, with its copies running ahead across units. So batches of any mixture of
// lengths load the machine evenly, and the grid does not depend on the lengths, which only the device knows. A run that ends
// inside a unit leaves a partial (O, m, l); those of a CTA's warps are joined in shared memory, those of several CTAs in
// scratch memory, always in the order of the keys, so results do not depend on timing.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "kv_cache.cuh"

namespace yk {

struct DecodeParams {
    PagedCache cache;
    const void * q;
    const void * gate;
    void * out;
    float * lse;
    const int32_t * lens;
    const int32_t * seq_ids;
    int32_t * status;
    int64_t q_row, q_head, out_row, out_head;  // elements
    int batch, heads, group, head_tiles, tile_heads;  // group: query heads per KV head; tiles of them, heads per tile
    int window, dtype;
    float scale_log2;  // softmax scale times log2 e
    float * partial;   // [CTAs][2][part floats]: a CTA's first and last unfinished unit
    int4 * joins;      // [CTAs] the unit that begins in the CTA and ends in a later one: x row, y unit of the row, z last CTA (-1: none)
    int min_tiles;     // tiles a warp takes at least
};

constexpr int DEC_TILE = 16;            // keys
constexpr float DEC_P_LOG2 = 14.0f;     // log2 of the factor that probabilities carry
constexpr int DEC_SMEM = 232448 - 1024; // dynamic shared memory of a CTA (the rest: the warps' records)

// ---- small helpers -------------------------------------------------------------------------------------------------

__device__ __forceinline__ void dec_mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dec_mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 transposition of 16-bit elements: lane (g, t) gives row g, columns 2t and 2t + 1, and receives row g of the transpose
__device__ __forceinline__ uint32_t dec_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t dec_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 dec_unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
__device__ __forceinline__ float dec_exp2(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int BYTES> __device__ __forceinline__ void dec_copy(uint32_t dst, const uint8_t * src, bool fill) {
    const int n = fill ? BYTES : 0;  // nothing copied: zeros
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void dec_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void dec_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 dec_lds4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 dec_lds2(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t dec_lds(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t dec_lds_u16(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void dec_sts(uint32_t at, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void dec_sts4(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// two E4M3 (the low or high half of a word) as f16 pairs
__device__ __forceinline__ uint32_t dec_e4m3(uint32_t two) {
    uint32_t h;
    asm volatile("{\n\t.reg .b16 x;\n\tcvt.u16.u32 x, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\t}" : "=r"(h) : "r"(two));
    return h;
}
// bytes 0 and 1 (PAIR 0) or 2 and 3 of x, unsigned with an offset of 128, as f16 pairs of the signed values: exact
template <int PAIR> __device__ __forceinline__ uint32_t dec_int8(uint32_t x) {
    const uint32_t h = __byte_perm(x, 0x64646464u, PAIR ? 0x4342 : 0x4140);  // 1024 + byte
    const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&h), __half2half2(__ushort_as_half((unsigned short)0x6480)));  // 1152
    return *reinterpret_cast<const uint32_t *>(&v);
}

// ---- layout --------------------------------------------------------------------------------------------------------

// FMT: format of the pools; NT: tiles of eight query heads; WIDE: q, gate and out are f32, and queries and probabilities enter
// the products as two parts (22 bits); otherwise f16 or bf16 and one part (11 bits, no less than such an output can tell).
template <int FMT, int HD, int NT, bool WIDE> struct DecodeShape {
    static constexpr bool IS_F32 = FMT == YUUKA_KV_F32, IS_Q8 = FMT == YUUKA_KV_Q8_0, IS_F8 = FMT == YUUKA_KV_F8;
    // lanes read what others have copied (Q8_0's words, F8's scales)
    static constexpr bool SHARED_COPIES = IS_Q8 || IS_F8;
    static constexpr int W = HD == 256 ? 4 : 8;  // warps: 256 dimensions leave a warp 128 registers of sums and queries
    static constexpr int COLS = 8 * NT, PARTS = WIDE ? 2 : 1;
    // Q8_0: words from key to key. K: 8 or 24 modulo 32, V: 4 or 12 modulo 16, which keeps the lanes' reads on different banks
    static constexpr int Q8_K = HD == 64 ? 24 : (HD == 128 ? 40 : 88), Q8_V = HD == 64 ? 20 : (HD == 128 ? 36 : 68);
    // F8: a lane's piece of V, 16 dimensions of 128 or 8 of 64; the scales of the tile's K and V lie behind K
    static constexpr int F8_V = HD == 64 ? 8 : 16;
    static constexpr int K_BYTES = IS_F32 ? HD * 64 : (IS_Q8 ? 64 * Q8_K : (IS_F8 ? HD * 16 + 128 : HD * 32));
    static constexpr int V_BYTES = IS_F32 ? HD * 64 : (IS_Q8 ? 64 * Q8_V : (IS_F8 ? HD * 16 : HD * 32));
    static constexpr int SLOT = (K_BYTES > V_BYTES ? K_BYTES : V_BYTES);
    static constexpr int PART_FLOATS = COLS * (HD + 2);
    static constexpr int PART_BYTES = (PART_FLOATS * 4 + 15) / 16 * 16;
    // queries in registers, or in shared memory where the sums leave too few (f32: 8 heads of all dimensions, split at use)
    static constexpr bool Q_SHARED = IS_F32 || HD / 4 * NT + HD / 8 * PARTS * NT > 128;
    static constexpr int Q_BYTES = !Q_SHARED ? 0 : (IS_F32 ? 8 * HD * 4 : COLS * HD * 2 * PARTS);
    static constexpr int WARP_BYTES = DEC_SMEM / W / 16 * 16;
    static constexpr int FIT = (WARP_BYTES - PART_BYTES - Q_BYTES) / SLOT;
    static constexpr int SLOTS = FIT > 8 ? 8 : FIT;  // K and V of a tile take one each
    static constexpr int AHEAD = SLOTS - 1;
    static constexpr int RING = SLOTS * SLOT;
    static_assert(SLOTS >= 2 && RING >= PART_BYTES, "a warp's shared memory");
    static constexpr int LAYOUT_BYTES = W * (RING + PART_BYTES + Q_BYTES);
    // accumulators: chunks of dimensions, DPL of them per lane
    static constexpr int DPL = (IS_F32 || IS_Q8) ? 4 : (IS_F8 ? F8_V : 8);
    static constexpr int CHUNKS = HD / (8 * DPL);

    // first of the two dimensions that rows g and g + 8 of product j of a chunk stand for
    __device__ static __forceinline__ int out_dim(int c, int j, int g) {
        if constexpr (IS_Q8) {
            // a block's words: an even block starts behind its scale with two values in word 0, so lane g has word g + 1
            return c * 32 + ((c & 1) ? 4 * g + 2 * j : (4 * g + 2 + 2 * j) & 31);
        } else {
            return c * 8 * DPL + g * DPL + 2 * j;
        }
    }
    // first of dimensions pair `half` (0, 1) that lane t multiplies in product m (16-bit products)
    __device__ static __forceinline__ int q_dim(int m, int half, int t) {
        if constexpr (IS_Q8) {
            const int blk = m >> 1, h = m & 1;
            return blk * 32 + ((blk & 1) ? 4 * (2 * t + h) + 2 * half : (4 * (1 + 2 * t + h) - 2 + 2 * half) & 31);
        } else if constexpr (IS_F8) {
            return 64 * (m >> 2) + 16 * t + 4 * (m & 3) + 2 * half;
        } else {
            return 32 * (m >> 1) + 8 * t + 4 * (m & 1) + 2 * half;
        }
    }
};

// ---- where a row's keys are ----------------------------------------------------------------------------------------

struct DecodeSpan {
    int first, end;  // keys of positions first .. end - 1
    int tiles;       // at least one, so that a row without keys is written too
    int seq;         // its sequence; -1: out of range
};
__host__ __device__ __forceinline__ DecodeSpan decode_span(const DecodeParams & p, int b, int & bad) {
    DecodeSpan s;
    const int n = kv_load(p.lens + b);
    s.seq = p.seq_ids ? kv_load(p.seq_ids + b) : b;
    bad = 0;
    if ((unsigned)s.seq >= (unsigned)p.cache.sequences) bad = KV_BAD_SEQUENCE;
    else if (n < 0 || n > p.cache.capacity) bad = KV_BAD_POSITION;
    s.end = bad ? 0 : n;
    s.first = p.window > 0 && s.end > p.window ? s.end - p.window : 0;
    s.tiles = s.end > s.first ? (s.end - s.first - 1) / DEC_TILE + 1 : 1;
    if (bad) s.seq = -1;
    return s;
}
__device__ __forceinline__ DecodeSpan decode_span(const DecodeParams & p, int b) {
    int bad;
    return decode_span(p, b, bad);
}

// A place in the sequence of tiles.
struct DecodeCursor {
    DecodeSpan span;
    int b, u, tile;
    __device__ __forceinline__ void next(const DecodeParams & p, int units) {
        if (++tile < span.tiles) return;
        tile = 0;
        if (++u < units) return;
        u = 0;
        if (++b < p.batch) span = decode_span(p, b);
    }
};

// ---- results -------------------------------------------------------------------------------------------------------

__device__ __forceinline__ float2 dec_read2(const void * base, int64_t at, int dtype) {
    if (dtype == YUUKA_DTYPE_F32) return *reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(base) + at);
    if (dtype == YUUKA_DTYPE_F16) return __half22float2(*reinterpret_cast<const __half2 *>(reinterpret_cast<const __half *>(base) + at));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(reinterpret_cast<const __nv_bfloat16 *>(base) + at));
}
// two neighbouring values of a head's result, gated and rounded to the output's type
__device__ __forceinline__ void dec_write2(const DecodeParams & p, int b, int head, int dim, float x, float y) {
    if (p.gate) {
        const float2 z = dec_read2(p.gate, b * p.q_row + head * p.q_head + dim, p.dtype);
        x *= 1.0f / (1.0f + expf(-z.x));
        y *= 1.0f / (1.0f + expf(-z.y));
    }
    const int64_t at = b * p.out_row + head * p.out_head + dim;
    if (p.dtype == YUUKA_DTYPE_F32) *reinterpret_cast<float2 *>(reinterpret_cast<float *>(p.out) + at) = make_float2(x, y);
    else if (p.dtype == YUUKA_DTYPE_F16) *reinterpret_cast<__half2 *>(reinterpret_cast<__half *>(p.out) + at) = __floats2half2_rn(x, y);
    else *reinterpret_cast<__nv_bfloat162 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + at) = __floats2bfloat162_rn(x, y);
}
__device__ __forceinline__ void dec_write_lse(const DecodeParams & p, int b, int head, float m, float l) {
    // (l carries the probabilities' factor)
    if (p.lse) p.lse[(int64_t)b * p.heads + head] = l == 0.0f ? -INFINITY : (m - DEC_P_LOG2 + log2f(l)) * 0.693147180559945309f;
}
// query heads of unit u of a row
struct DecodeHeads {
    int kv_head, first, count;
};
__device__ __forceinline__ DecodeHeads decode_heads(const DecodeParams & p, int u) {
    DecodeHeads h;
    h.kv_head = u / p.head_tiles;
    const int ht = u - h.kv_head * p.head_tiles;
    h.first = h.kv_head * p.group + ht * p.tile_heads;
    h.count = min(p.tile_heads, p.group - ht * p.tile_heads);
    return h;
}

// A chain of partials of one unit, `count` of them `stride` floats apart from `second` on, joined and written: as the unit's
// result (final), or as one partial. Threads of a CTA take pairs of dimensions.
template <int HD, int COLS>
__device__ __forceinline__ void dec_join(const DecodeParams & p, const float * head, const float * second, int stride, int count, bool final,
                                         int b, int u, float * dst, int thread, int threads) {
    const DecodeHeads h = decode_heads(p, u);
    for (int i = thread; i < COLS * HD / 2; i += threads) {
        const int col = i / (HD / 2), dim = 2 * (i - col * (HD / 2));
        if (col >= h.count) continue;
        float m = -INFINITY;
        for (int k = 0; k < count; k++) m = fmaxf(m, (k ? second + (size_t)(k - 1) * stride : head)[COLS * HD + col]);
        float l = 0.0f, x = 0.0f, y = 0.0f;
        for (int k = 0; k < count; k++) {
            const float * part = k ? second + (size_t)(k - 1) * stride : head;
            const float f = exp2f(part[COLS * HD + col] - m);
            const float2 o = *reinterpret_cast<const float2 *>(part + col * HD + dim);
            l = fmaf(f, part[COLS * HD + COLS + col], l);
            x = fmaf(f, o.x, x);
            y = fmaf(f, o.y, y);
        }
        if (final) {
            dec_write2(p, b, h.first + col, dim, x / l, y / l);
            if (dim == 0) dec_write_lse(p, b, h.first + col, m, l);
        } else {
            *reinterpret_cast<float2 *>(dst + col * HD + dim) = make_float2(x, y);
            if (dim == 0) {
                dst[COLS * HD + col] = m;
                dst[COLS * HD + COLS + col] = l;
            }
        }
    }
}

// ---- the kernel ----------------------------------------------------------------------------------------------------

template <int FMT, int HD, int NT, bool WIDE>
__global__ void __launch_bounds__(DecodeShape<FMT, HD, NT, WIDE>::W * 32, 1) attention_decode_kernel(const DecodeParams p) {
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    constexpr int W = S::W, COLS = S::COLS, SLOTS = S::SLOTS, AHEAD = S::AHEAD, CHUNKS = S::CHUNKS, DPL = S::DPL;
    extern __shared__ __align__(16) uint8_t smem[];
    // What the CTA's warps leave unfinished: a unit begun by an earlier warp (head: 1 it ends here, 2 it goes on), a unit begun
    // here (tail: 1) that goes on
    __shared__ int head_kind[W], tail_kind[W], head_b[W], head_u[W], tail_b[W], tail_u[W];
    __shared__ long long tail_end[W];  // tile behind the tail's unit
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t * const ring_at = smem + warp * S::RING;
    float * const head_part = reinterpret_cast<float *>(smem + W * S::RING + warp * S::PART_BYTES);
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_at);
    const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(smem + W * (S::RING + S::PART_BYTES) + warp * S::Q_BYTES) + lane * 16;
    pdl_entry();

    // this warp's run of tiles
    const int units = p.cache.kv_heads * p.head_tiles;
    long long total = 0;
    for (int b = lane; b < p.batch; b += 32) {
        int bad;
        total += decode_span(p, b, bad).tiles;
        if (bad && p.status && blockIdx.x == 0 && warp == 0) atomicOr(p.status, bad);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= units;
    const long long warps = (long long)gridDim.x * W;
    const long long share = max((long long)p.min_tiles, (total + warps - 1) / warps);
    const long long begin = ((long long)blockIdx.x * W + warp) * share;
    const int count = begin < total ? (int)min(share, total - begin) : 0;

    if (lane == 0) head_kind[warp] = tail_kind[warp] = 0;
    if (count > 0) {
        DecodeCursor use;
        {
            long long before = 0;
            int base = 0;
            use.b = 0;
            for (; base < p.batch; base += 32) {  // (begin < total: some row holds it)
                const int b = base + lane;
                const long long mine = b < p.batch ? (long long)decode_span(p, b).tiles * units : 0;
                long long sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long v = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += v;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, before + sum > begin);
                if (hit) {
                    const int at = __ffs(hit) - 1;
                    use.b = base + at;
                    before += __shfl_sync(0xffffffffu, sum - mine, at);
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
            use.span = decode_span(p, use.b);
            const long long rest = begin - before;
            use.u = min((int)(rest / use.span.tiles), units - 1);  // (it is less, unless lengths change under the call)
            use.tile = (int)(rest - (long long)use.u * use.span.tiles);
        }

        // -- copies: `ahead` is the tile whose K or V is fetched next, `slot_row` the pool row of its key lane % 16 (-1: no
        // key there, zeros; -2: a bad block, NaN)
        DecodeCursor ahead = use;
        int fetched = 0;  // tiles of the run whose V has been asked for
        int slot_row = -1;
        const int64_t head_bytes = FMT == YUUKA_KV_F32 ? HD * 4 : (FMT == YUUKA_KV_F16 ? HD * 2 : (FMT == YUUKA_KV_Q8_0 ? HD / 32 * 34 : HD));
        int64_t head_at = 0;
        auto look_up = [&] {
            const int pos = ahead.span.first + ahead.tile * DEC_TILE + (lane & 15);
            slot_row = -1;
            if (pos < ahead.span.end) {
                slot_row = kv_slot(p.cache, p.cache.tables + (int64_t)ahead.span.seq * p.cache.table_stride, pos);
                if (slot_row == -2 && p.status) atomicOr(p.status, KV_BAD_BLOCK);
            }
            head_at = (int64_t)(ahead.u / p.head_tiles) * head_bytes;
        };
        look_up();
        auto row_of = [&](const uint8_t * pool, int key, int & row) {
            row = __shfl_sync(0xffffffffu, slot_row, key);
            return pool + (int64_t)max(row, 0) * p.cache.row_bytes + head_at;
        };
        auto fetch = [&](auto is_v, int slot) {
            constexpr bool V = decltype(is_v)::value;
            const uint8_t * pool = V ? p.cache.v : p.cache.k;
            const uint32_t base = ring + slot * S::SLOT;
            if (fetched < count) {
                if constexpr (FMT == YUUKA_KV_Q8_0) {
                    constexpr int WORDS = HD / 32 * 34 / 4;
                    const int l8 = lane & 7;
#pragma unroll
                    for (int kg = 0; kg < 4; kg++) {
                        const int key = 4 * kg + (lane >> 3);
                        int row;
                        const uint8_t * src = row_of(pool, key, row) + 4 * l8;
                        const uint32_t dst = base + 4 * (V ? key * S::Q8_V : key * S::Q8_K + 1) + 4 * l8;
#pragma unroll
                        for (int i = 0; i < (WORDS + 7) / 8; i++) {
                            const int w = 8 * i + l8;
                            // K: one word between the pairs of blocks (17 words), so that lanes read two aligned words
                            const int gap = V ? 0 : (w >= 17) + (w >= 34) + (w >= 51);
                            if (w < WORDS) {
                                if (row == -2) dec_sts(dst + 32 * i + 4 * gap, 0xffffffffu);
                                else dec_copy<4>(dst + 32 * i + 4 * gap, src + 32 * i, row >= 0);
                            }
                        }
                    }
                } else if constexpr (!V) {
                    constexpr int PIECES = S::K_BYTES / 1024;  // 16 bytes of keys g and g + 8, per lane
                    int r0, r1;
                    const uint8_t * s0 = row_of(pool, g, r0) + 16 * t;
                    const uint8_t * s1 = row_of(pool, g + 8, r1) + 16 * t;
                    const uint32_t dst = base + lane * 16;
#pragma unroll
                    for (int i = 0; i < PIECES; i++) {
                        if (r0 != -2) dec_copy<16>(dst + 1024 * i, s0 + 64 * i, r0 >= 0);
                        else dec_sts4(dst + 1024 * i, make_uint4(~0u, ~0u, ~0u, ~0u));
                        if (r1 != -2) dec_copy<16>(dst + 1024 * i + 512, s1 + 64 * i, r1 >= 0);
                        else dec_sts4(dst + 1024 * i + 512, make_uint4(~0u, ~0u, ~0u, ~0u));
                    }
                    if constexpr (FMT == YUUKA_KV_F8) {
                        // scales: lanes 0-15 of K, 16-31 of V
                        const int kv_head = ahead.u / p.head_tiles;
                        const uint8_t * src = (lane < 16 ? p.cache.k : p.cache.v) + (int64_t)max(slot_row, 0) * p.cache.row_bytes +
                                              (int64_t)p.cache.kv_heads * HD + 4 * kv_head;
                        if (slot_row == -2) dec_sts(base + HD * 16 + 4 * lane, 0x7fffffffu);
                        else dec_copy<4>(base + HD * 16 + 4 * lane, src, slot_row >= 0);
                    }
                } else {
                    constexpr int PIECE = FMT == YUUKA_KV_F8 ? S::F8_V : 16;  // a lane's bytes of keys 2t, 2t + 1, 2t + 8, 2t + 9
                    constexpr int PIECES = S::V_BYTES / (128 * PIECE);
                    const uint32_t dst = base + lane * PIECE;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        int row;
                        const uint8_t * src = row_of(pool, 2 * t + (k & 1) + 8 * (k >> 1), row) + PIECE * g;
#pragma unroll
                        for (int i = 0; i < PIECES; i++) {
                            const uint32_t to = dst + (i * 4 + k) * 32 * PIECE;
                            if (row != -2) dec_copy<PIECE>(to, src + 8 * PIECE * i, row >= 0);
                            else
                                for (int w = 0; w < PIECE; w += 4) dec_sts(to + w, ~0u);
                        }
                    }
                }
                if constexpr (V) {
                    fetched++;
                    if (fetched < count) {
                        ahead.next(p, units);
                        look_up();
                    }
                }
            }
            dec_commit();
        };
        int put = 0;  // slot that is filled next
        auto fetch_next = [&](auto is_v) {
            fetch(is_v, put);
            put = put + 1 == SLOTS ? 0 : put + 1;
        };
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (i & 1) fetch_next(std::true_type());
            else fetch_next(std::false_type());
        }

        // -- per unit: queries, statistics and sums
        constexpr int QM = HD / 16;  // 16-bit products over the head dimension
        uint32_t q[S::Q_SHARED ? 1 : NT][S::Q_SHARED ? 1 : S::PARTS][S::Q_SHARED ? 1 : QM][2];
        float scale[NT][2];          // of the columns' scores
        float m[NT][2], l[NT][2];    // l: of this lane's keys
        float o[NT][CHUNKS][DPL / 2][4];
        float v_scale = 1.0f;        // Q8_0, F8: o is in units of it (a power of two)
        bool from_start = false;

        auto load_queries = [&] {
            const DecodeHeads h = decode_heads(p, use.u);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int col = nt * 8 + g;
                const bool has = col < h.count;
                const int64_t at = use.b * p.q_row + (h.first + (has ? col : 0)) * p.q_head;
                if constexpr (S::IS_F32) {
                    // dimensions 16 i + 4 t .. + 3 of head g
#pragma unroll 4
                    for (int i = 0; i < HD / 16; i++) {
                        const float2 x = has ? dec_read2(p.q, at + 16 * i + 4 * t, p.dtype) : make_float2(0.f, 0.f);
                        const float2 y = has ? dec_read2(p.q, at + 16 * i + 4 * t + 2, p.dtype) : make_float2(0.f, 0.f);
                        dec_sts4(q_at + 512 * i, make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y)));
                    }
                    scale[nt][0] = scale[nt][1] = p.scale_log2;
                } else {
                    // scaled to a largest magnitude of 2^14 .. 2^15, so that two f16 parts hold 22 bits of what matters
                    float amax = 0.0f;
#pragma unroll 4
                    for (int i = 0; i < 2 * QM; i++) {
                        const float2 x = has ? dec_read2(p.q, at + S::q_dim(i >> 1, i & 1, t), p.dtype) : make_float2(0.f, 0.f);
                        amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
                    }
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    const int e = min(max((int)(__float_as_uint(amax) >> 23), 15), 254);
                    const float up = __int_as_float((268 - e) << 23);                        // 2^(14 - (e - 127))
                    const float down = p.scale_log2 * __int_as_float((e - 14) << 23);        // scale / up
                    scale[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
                    scale[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
                    for (int i = 0; i < QM; i++) {
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            float2 x = has ? dec_read2(p.q, at + S::q_dim(i, half, t), p.dtype) : make_float2(0.f, 0.f);
                            x.x *= up;
                            x.y *= up;
                            hi[half] = dec_pack(x.x, x.y);
                            const float2 r = dec_unpack(hi[half]);
                            lo[half] = dec_pack(x.x - r.x, x.y - r.y);
                        }
                        if constexpr (S::Q_SHARED) {
                            if constexpr (WIDE) dec_sts4(q_at + 512 * (nt * QM + i), make_uint4(hi[0], hi[1], lo[0], lo[1]));
                            else asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(q_at - 8 * lane + 256 * (nt * QM + i)), "r"(hi[0]), "r"(hi[1]) : "memory");
                        } else {
                            q[nt][0][i][0] = hi[0];
                            q[nt][0][i][1] = hi[1];
                            if constexpr (WIDE) {
                                q[nt][1][i][0] = lo[0];
                                q[nt][1][i][1] = lo[1];
                            }
                        }
                    }
                }
            }
        };
        // fragments of product i of the head dimension: part 0 in x, y, part 1 in z, w
        auto query = [&](int nt, int i) {
            uint4 f = make_uint4(0, 0, 0, 0);
            if constexpr (S::Q_SHARED) {
                if constexpr (WIDE) f = dec_lds4(q_at + 512 * (nt * QM + i));
                else {
                    const uint2 r = dec_lds2(q_at - 8 * lane + 256 * (nt * QM + i));
                    f.x = r.x;
                    f.y = r.y;
                }
            } else {
                f.x = q[nt][0][i][0];
                f.y = q[nt][0][i][1];
                if constexpr (WIDE) {
                    f.z = q[nt][1][i][0];
                    f.w = q[nt][1][i][1];
                }
            }
            return f;
        };
        auto rescale = [&](const float (&f)[NT][2]) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                    for (int j = 0; j < DPL / 2; j++) {
                        o[nt][c][j][0] *= f[nt][0];
                        o[nt][c][j][1] *= f[nt][1];
                        o[nt][c][j][2] *= f[nt][0];
                        o[nt][c][j][3] *= f[nt][1];
                    }
        };
        // The largest scale of V among the tile's keys (bits of its magnitude) joins the unit of o; returns the unit's inverse.
        auto take_v_scale = [&](uint32_t bits) {
            bits = __reduce_max_sync(0xffffffffu, bits);
            // the next power of two; 2^-126 at least, and a NaN stays one
            const uint32_t top = bits >= 0x7f000000u ? bits : max((bits + 0x7fffffu) & 0x7f800000u, 0x00800000u);
            const float v = __uint_as_float(top);
            if (!(v <= v_scale)) {  // (uniform)
                float f[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) f[nt][0] = f[nt][1] = v_scale / v;
                rescale(f);
                v_scale = v;
            }
            return 1.0f / v_scale;
        };

        int take = 0;  // slot that is used next
        for (int it = 0; it < count; it++) {
            // ---- K: scores
            dec_wait<AHEAD - 1>();
            if constexpr (S::SHARED_COPIES) __syncwarp();
            if constexpr (AHEAD & 1) fetch_next(std::true_type());
            else fetch_next(std::false_type());
            const uint32_t ks = ring + take * S::SLOT;
            take = take + 1 == SLOTS ? 0 : take + 1;

            if (it == 0 || use.tile == 0) {
                from_start = use.tile == 0;
                load_queries();
                v_scale = __uint_as_float(0x00800000u);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    m[nt][0] = m[nt][1] = -INFINITY;
                    l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                        for (int j = 0; j < DPL / 2; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[nt][c][j][e] = 0.0f;
                }
                // a row that is out of range: everything becomes NaN
                if (use.span.seq < 0)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) l[nt][0] = l[nt][1] = __uint_as_float(0x7fffffffu);
            }
            const int keys = min(DEC_TILE, use.span.end - use.span.first - use.tile * DEC_TILE);  // 0 for a row without any

            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[nt][e] = 0.0f;
            if constexpr (S::IS_F32) {
                // three products of tf32 parts: hi hi, hi lo, lo hi
                float s2[NT][4] = {};
#pragma unroll
                for (int c = 0; c < HD / 16; c++) {
                    const uint4 ka = dec_lds4(ks + lane * 16 + 1024 * c), kb = dec_lds4(ks + lane * 16 + 1024 * c + 512);
                    const uint4 f = dec_lds4(q_at + 512 * c);
                    const uint32_t a[8] = {ka.x, kb.x, ka.y, kb.y, ka.z, kb.z, ka.w, kb.w};
                    const uint32_t b[4] = {f.x, f.y, f.z, f.w};
                    uint32_t ah[8], al[8], bh[4], bl[4];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        ah[i] = a[i] & 0xffffe000u;
                        al[i] = __float_as_uint(__uint_as_float(a[i]) - __uint_as_float(ah[i]));
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        bh[i] = b[i] & 0xffffe000u;
                        bl[i] = __float_as_uint(__uint_as_float(b[i]) - __uint_as_float(bh[i]));
                    }
                    dec_mma8(s[0], ah[0], ah[1], ah[2], ah[3], bh[0], bh[1]);
                    dec_mma8(s2[0], ah[4], ah[5], ah[6], ah[7], bh[2], bh[3]);
                    dec_mma8(s[0], al[0], al[1], al[2], al[3], bh[0], bh[1]);
                    dec_mma8(s2[0], al[4], al[5], al[6], al[7], bh[2], bh[3]);
                    if constexpr (WIDE) {  // (16-bit queries have no second part)
                        dec_mma8(s[0], ah[0], ah[1], ah[2], ah[3], bl[0], bl[1]);
                        dec_mma8(s2[0], ah[4], ah[5], ah[6], ah[7], bl[2], bl[3]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[0][e] += s2[0][e];
            } else if constexpr (S::IS_Q8) {
                const uint32_t ka = ks + 4 * (g * S::Q8_K + 1), kb = ka + 32 * S::Q8_K;  // keys g and g + 8
#pragma unroll
                for (int pair = 0; pair < HD / 64; pair++) {
                    uint32_t w[2][4];   // [key][word]: two of the even block, two of the odd one
                    float d[2][2];      // [key][block]
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t at = (k ? kb : ka) + 72 * pair;
                        const uint2 even = dec_lds2(at + 4 * (1 + 2 * t)), odd = dec_lds2(at + 4 * (9 + 2 * t));
                        const uint32_t w0 = dec_lds(at), w8 = dec_lds(at + 32);
                        d[k][0] = __half2float(__ushort_as_half((unsigned short)w0));
                        d[k][1] = __half2float(__ushort_as_half((unsigned short)(w8 >> 16)));
                        w[k][0] = even.x ^ 0x80808080u;
                        // word 8 is the block's last two values and the next scale: its first two are in word 0
                        w[k][1] = (t == 3 ? __byte_perm(w8, w0, 0x7610) : even.y) ^ 0x80808080u;
                        w[k][2] = odd.x ^ 0x80808080u;
                        w[k][3] = odd.y ^ 0x80808080u;
                    }
#pragma unroll
                    for (int blk = 0; blk < 2; blk++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t u0 = w[0][2 * blk + h], u1 = w[1][2 * blk + h];
                                const uint32_t a0 = dec_int8<0>(u0), a1 = dec_int8<0>(u1), a2 = dec_int8<1>(u0), a3 = dec_int8<1>(u1);
                                const uint4 f = query(nt, 4 * pair + 2 * blk + h);
                                dec_mma16(x, a0, a1, a2, a3, f.x, f.y);
                                if constexpr (WIDE) dec_mma16(x, a0, a1, a2, a3, f.z, f.w);
                            }
                            s[nt][0] = fmaf(x[0], d[0][blk], s[nt][0]);
                            s[nt][1] = fmaf(x[1], d[0][blk], s[nt][1]);
                            s[nt][2] = fmaf(x[2], d[1][blk], s[nt][2]);
                            s[nt][3] = fmaf(x[3], d[1][blk], s[nt][3]);
                        }
                }
            } else {
                float s2[NT][4] = {};
                if constexpr (S::IS_F8) {
#pragma unroll
                    for (int c = 0; c < HD / 64; c++) {
                        const uint4 ka = dec_lds4(ks + lane * 16 + 1024 * c), kb = dec_lds4(ks + lane * 16 + 1024 * c + 512);
                        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t a0 = dec_e4m3(wa[i]), a1 = dec_e4m3(wb[i]), a2 = dec_e4m3(wa[i] >> 16), a3 = dec_e4m3(wb[i] >> 16);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const uint4 f = query(nt, 4 * c + i);
                                dec_mma16((i & 1) ? s2[nt] : s[nt], a0, a1, a2, a3, f.x, f.y);
                                if constexpr (WIDE) dec_mma16((i & 1) ? s2[nt] : s[nt], a0, a1, a2, a3, f.z, f.w);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < HD / 32; c++) {
                        const uint4 ka = dec_lds4(ks + lane * 16 + 1024 * c), kb = dec_lds4(ks + lane * 16 + 1024 * c + 512);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint4 f = query(nt, 2 * c), f2 = query(nt, 2 * c + 1);
                            dec_mma16(s[nt], ka.x, kb.x, ka.y, kb.y, f.x, f.y);
                            dec_mma16(s2[nt], ka.z, kb.z, ka.w, kb.w, f2.x, f2.y);
                            if constexpr (WIDE) {
                                dec_mma16(s[nt], ka.x, kb.x, ka.y, kb.y, f.z, f.w);
                                dec_mma16(s2[nt], ka.z, kb.z, ka.w, kb.w, f2.z, f2.w);
                            }
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[nt][e] += s2[nt][e];
            }
            float vd[2] = {1.0f, 1.0f};  // F8: scales of V of keys g and g + 8
            if constexpr (S::IS_F8) {
                const float d0 = __uint_as_float(dec_lds(ks + HD * 16 + 4 * g)), d1 = __uint_as_float(dec_lds(ks + HD * 16 + 4 * (g + 8)));
                vd[0] = __uint_as_float(dec_lds(ks + HD * 16 + 64 + 4 * g));
                vd[1] = __uint_as_float(dec_lds(ks + HD * 16 + 64 + 4 * (g + 8)));
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s[nt][0] *= d0;
                    s[nt][1] *= d0;
                    s[nt][2] *= d1;
                    s[nt][3] *= d1;
                }
            }

            // ---- running maximum and sum; s becomes the probabilities of keys g (0, 1) and g + 8 (2, 3), columns 2t and 2t + 1
            if (keys > 0) {  // (uniform)
                float corr[NT][2];
                bool moved = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) s[nt][e] = (g + 8 * (e >> 1) < keys) ? s[nt][e] * scale[nt][e & 1] : -INFINITY;
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float mx = fmaxf(s[nt][c], s[nt][c + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float top = fmaxf(m[nt][c], mx);
                        corr[nt][c] = dec_exp2(m[nt][c] - top);
                        moved |= top > m[nt][c];
                        m[nt][c] = top;
                        s[nt][c] = dec_exp2(s[nt][c] - top + DEC_P_LOG2);
                        s[nt][c + 2] = dec_exp2(s[nt][c + 2] - top + DEC_P_LOG2);
                        l[nt][c] = fmaf(l[nt][c], corr[nt][c], s[nt][c] + s[nt][c + 2]);
                    }
                }
                if (__any_sync(0xffffffffu, moved)) rescale(corr);
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[nt][e] = 0.0f;
            }
            // probabilities as fragments: keys become the dimension that is summed over
            uint32_t pb[NT][S::PARTS][2];
            auto fragments = [&](float f0, float f1) {  // with factors of keys g and g + 8
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float x0 = s[nt][0] * f0, x1 = s[nt][1] * f0, y0 = s[nt][2] * f1, y1 = s[nt][3] * f1;
                    const uint32_t hx = dec_pack(x0, x1), hy = dec_pack(y0, y1);
                    pb[nt][0][0] = dec_transpose(hx);
                    pb[nt][0][1] = dec_transpose(hy);
                    if constexpr (WIDE) {
                        const float2 rx = dec_unpack(hx), ry = dec_unpack(hy);
                        pb[nt][1][0] = dec_transpose(dec_pack(x0 - rx.x, x1 - rx.y));
                        pb[nt][1][1] = dec_transpose(dec_pack(y0 - ry.x, y1 - ry.y));
                    }
                }
            };
            if constexpr (FMT == YUUKA_KV_F16) fragments(1.0f, 1.0f);
            else if constexpr (S::IS_F8) {
                const float inv = take_v_scale(max(__float_as_uint(fabsf(vd[0])), __float_as_uint(fabsf(vd[1]))));
                fragments(vd[0] * inv, vd[1] * inv);
            }

            // ---- V: sums
            dec_wait<AHEAD - 1>();
            if constexpr (S::SHARED_COPIES) __syncwarp();
            if constexpr (AHEAD & 1) fetch_next(std::false_type());
            else fetch_next(std::true_type());
            const uint32_t vs = ring + take * S::SLOT;
            take = take + 1 == SLOTS ? 0 : take + 1;

            if constexpr (S::IS_F32) {
                // probabilities in f32 change hands as two 16-bit halves; lane (g, t) then has keys 2t, 2t + 1 (and + 8) of column g
                float pk[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t x = __float_as_uint(s[0][2 * h]), y = __float_as_uint(s[0][2 * h + 1]);
                    const uint32_t low = dec_transpose(__byte_perm(x, y, 0x5410)), high = dec_transpose(__byte_perm(x, y, 0x7632));
                    pk[2 * h] = __uint_as_float(__byte_perm(low, high, 0x5410));
                    pk[2 * h + 1] = __uint_as_float(__byte_perm(low, high, 0x7632));
                }
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    ph[i] = __float_as_uint(pk[i]) & 0xffffe000u;
                    pl[i] = __float_as_uint(pk[i] - __uint_as_float(ph[i]));
                }
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    uint32_t v[4][4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint4 r = dec_lds4(vs + lane * 16 + (c * 4 + k) * 512);
                        v[k][0] = r.x; v[k][1] = r.y; v[k][2] = r.z; v[k][3] = r.w;
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t a[4] = {v[2 * h][2 * j], v[2 * h][2 * j + 1], v[2 * h + 1][2 * j], v[2 * h + 1][2 * j + 1]};
                            uint32_t ah[4], al[4];
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                ah[i] = a[i] & 0xffffe000u;
                                al[i] = __float_as_uint(__uint_as_float(a[i]) - __uint_as_float(ah[i]));
                            }
                            dec_mma8(o[0][c][j], ah[0], ah[1], ah[2], ah[3], ph[2 * h], ph[2 * h + 1]);
                            dec_mma8(o[0][c][j], al[0], al[1], al[2], al[3], ph[2 * h], ph[2 * h + 1]);
                            dec_mma8(o[0][c][j], ah[0], ah[1], ah[2], ah[3], pl[2 * h], pl[2 * h + 1]);
                        }
                }
            } else if constexpr (S::IS_Q8) {
                // scales of V: of keys g and g + 8, block by block, into the probabilities
                const uint32_t va = vs + 4 * g * S::Q8_V, vb = va + 32 * S::Q8_V;
                float d[2][HD / 32];
                uint32_t top = 0;
#pragma unroll
                for (int blk = 0; blk < HD / 32; blk++) {
                    const uint32_t x = dec_lds_u16(va + 34 * blk), y = dec_lds_u16(vb + 34 * blk);
                    d[0][blk] = __half2float(__ushort_as_half((unsigned short)x));
                    d[1][blk] = __half2float(__ushort_as_half((unsigned short)y));
                    top = max(top, max(__float_as_uint(fabsf(d[0][blk])), __float_as_uint(fabsf(d[1][blk]))));
                }
                const float inv = take_v_scale(top);
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    fragments(d[0][c] * inv, d[1][c] * inv);
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t at = vs + 4 * (2 * t + (k & 1) + 8 * (k >> 1)) * S::Q8_V + 68 * (c >> 1);
                        if (c & 1) w[k] = dec_lds(at + 4 * (9 + g));
                        else {
                            const uint32_t x = dec_lds(at + 4 * (1 + g)), w0 = dec_lds(at);
                            w[k] = g == 7 ? __byte_perm(x, w0, 0x7610) : x;
                        }
                        w[k] ^= 0x80808080u;
                    }
                    const uint32_t x01 = __byte_perm(w[0], w[1], 0x5140), x23 = __byte_perm(w[0], w[1], 0x7362);
                    const uint32_t y01 = __byte_perm(w[2], w[3], 0x5140), y23 = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t x = j ? x23 : x01, y = j ? y23 : y01;
                        const uint32_t a0 = dec_int8<0>(x), a1 = dec_int8<1>(x), a2 = dec_int8<0>(y), a3 = dec_int8<1>(y);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            dec_mma16(o[nt][c][j], a0, a1, a2, a3, pb[nt][0][0], pb[nt][0][1]);
                            if constexpr (WIDE) dec_mma16(o[nt][c][j], a0, a1, a2, a3, pb[nt][1][0], pb[nt][1][1]);
                        }
                    }
                }
            } else if constexpr (S::IS_F8) {
                constexpr int WORDS = S::F8_V / 4;
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    uint32_t v[4][WORDS];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t at = vs + lane * S::F8_V + (c * 4 + k) * 32 * S::F8_V;
                        if constexpr (WORDS == 4) {
                            const uint4 r = dec_lds4(at);
                            v[k][0] = r.x; v[k][1] = r.y; v[k][2] = r.z; v[k][3] = r.w;
                        } else {
                            const uint2 r = dec_lds2(at);
                            v[k][0] = r.x; v[k][1] = r.y;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < WORDS; w++) {
                        // bytes of two keys next to one another: values of one dimension
                        const uint32_t x01 = __byte_perm(v[0][w], v[1][w], 0x5140), x23 = __byte_perm(v[0][w], v[1][w], 0x7362);
                        const uint32_t y01 = __byte_perm(v[2][w], v[3][w], 0x5140), y23 = __byte_perm(v[2][w], v[3][w], 0x7362);
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t x = j ? x23 : x01, y = j ? y23 : y01;
                            const uint32_t a0 = dec_e4m3(x), a1 = dec_e4m3(x >> 16), a2 = dec_e4m3(y), a3 = dec_e4m3(y >> 16);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                dec_mma16(o[nt][c][2 * w + j], a0, a1, a2, a3, pb[nt][0][0], pb[nt][0][1]);
                                if constexpr (WIDE) dec_mma16(o[nt][c][2 * w + j], a0, a1, a2, a3, pb[nt][1][0], pb[nt][1][1]);
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    uint32_t v[4][4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint4 r = dec_lds4(vs + lane * 16 + (c * 4 + k) * 512);
                        v[k][0] = r.x; v[k][1] = r.y; v[k][2] = r.z; v[k][3] = r.w;
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t a0 = __byte_perm(v[0][j], v[1][j], 0x5410), a1 = __byte_perm(v[0][j], v[1][j], 0x7632);
                        const uint32_t a2 = __byte_perm(v[2][j], v[3][j], 0x5410), a3 = __byte_perm(v[2][j], v[3][j], 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            dec_mma16(o[nt][c][j], a0, a1, a2, a3, pb[nt][0][0], pb[nt][0][1]);
                            if constexpr (WIDE) dec_mma16(o[nt][c][j], a0, a1, a2, a3, pb[nt][1][0], pb[nt][1][1]);
                        }
                    }
                }
            }

            // ---- the end of the unit or of the run
            const bool ends = use.tile + 1 == use.span.tiles;
            if (ends || it + 1 == count) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
                        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
                        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
                    }
                if constexpr (!S::IS_Q8 && !S::IS_F8) v_scale = 1.0f;
                if (ends && from_start) {
                    const DecodeHeads h = decode_heads(p, use.u);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int col = nt * 8 + 2 * t + e;
                            if (col >= h.count) continue;
                            const float inv = l[nt][e] == 0.0f ? 0.0f : v_scale / l[nt][e];
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                for (int j = 0; j < DPL / 2; j++)
                                    dec_write2(p, use.b, h.first + col, S::out_dim(c, j, g), o[nt][c][j][e] * inv, o[nt][c][j][e + 2] * inv);
                            if (g == 0) dec_write_lse(p, use.b, h.first + col, m[nt][e], l[nt][e]);
                        }
                } else {
                    // a unit begun earlier goes to its own place; one begun here is the run's last, and its ring is done with
                    // once every lane has used its copies
                    float * part = head_part;
                    if (from_start) {
                        dec_wait<0>();
                        __syncwarp();
                        part = reinterpret_cast<float *>(ring_at);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int col = nt * 8 + 2 * t + e;
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                for (int j = 0; j < DPL / 2; j++)
                                    *reinterpret_cast<float2 *>(part + col * HD + S::out_dim(c, j, g)) =
                                        make_float2(o[nt][c][j][e] * v_scale, o[nt][c][j][e + 2] * v_scale);
                            if (g == 0) {
                                part[COLS * HD + col] = m[nt][e];
                                part[COLS * HD + COLS + col] = l[nt][e];
                            }
                        }
                    if (lane == 0) {
                        if (from_start) {
                            tail_kind[warp] = 1;
                            tail_b[warp] = use.b;
                            tail_u[warp] = use.u;
                            tail_end[warp] = begin + it + (use.span.tiles - use.tile);
                        } else {
                            head_kind[warp] = ends ? 1 : 2;
                            head_b[warp] = use.b;
                            head_u[warp] = use.u;
                        }
                    }
                }
            }
            use.next(p, units);
        }
        dec_wait<0>();
    }

    // ---- joining the warps' partials, in the order of the keys
    __syncthreads();
    auto head_of = [&](int w) { return reinterpret_cast<float *>(smem + W * S::RING + w * S::PART_BYTES); };
    float * const cta_head = p.partial + (size_t)blockIdx.x * 2 * S::PART_FLOATS;
    float * const cta_tail = cta_head + S::PART_FLOATS;
    int join_b = 0, join_u = 0, join_last = -1;
    if (head_kind[0]) {
        int n = 1;
        bool ends = head_kind[0] == 1;
        while (!ends && n < W && head_kind[n]) ends = head_kind[n++] == 1;
        // (warp 0 of CTA 0 never begins inside a unit)
        dec_join<HD, COLS>(p, head_of(0), head_of(1), S::PART_BYTES / 4, n, false, head_b[0], head_u[0], cta_head, threadIdx.x, W * 32);
    }
    for (int w = 0; w < W; w++) {
        if (!tail_kind[w]) continue;
        int n = 1;
        bool ends = false;
        while (!ends && w + n < W && head_kind[w + n]) ends = head_kind[w + n++] == 1;
        dec_join<HD, COLS>(p, reinterpret_cast<const float *>(smem + w * S::RING), w + 1 < W ? head_of(w + 1) : nullptr, S::PART_BYTES / 4, n, ends,
                           tail_b[w], tail_u[w], cta_tail, threadIdx.x, W * 32);
        if (!ends) {
            join_b = tail_b[w];
            join_u = tail_u[w];
            join_last = (int)((tail_end[w] - 1) / (share * W));
        }
    }
    if (threadIdx.x == 0) p.joins[blockIdx.x] = make_int4(join_b, join_u, join_last, 0);
}

// The units that several CTAs share: a CTA per (CTA in which such a unit begins, column).
template <int HD, int COLS> __global__ void __launch_bounds__(HD / 2) attention_decode_join_kernel(const DecodeParams p) {
    constexpr int PART = COLS * (HD + 2);
    pdl_entry();
    const int c = blockIdx.x, col = blockIdx.y;
    const int4 join = p.joins[c];
    if (join.z < 0) return;
    const DecodeHeads h = decode_heads(p, join.y);
    if (col >= h.count) return;
    const int n = join.z - c + 1;  // partials: the tail of CTA c and the heads of the following ones
    const float * tail = p.partial + ((size_t)c * 2 + 1) * PART;
    const float * heads = p.partial + (size_t)(c + 1) * 2 * PART;
    auto part = [&](int k) { return k ? heads + (size_t)(k - 1) * 2 * PART : tail; };
    float m = -INFINITY;
    for (int k = 0; k < n; k++) m = fmaxf(m, part(k)[COLS * HD + col]);
    float l = 0.0f, x = 0.0f, y = 0.0f;
    const int dim = 2 * threadIdx.x;
#pragma unroll 8
    for (int k = 0; k < n; k++) {
        const float * q = part(k);
        const float f = exp2f(q[COLS * HD + col] - m);
        const float2 o = *reinterpret_cast<const float2 *>(q + col * HD + dim);
        l = fmaf(f, q[COLS * HD + COLS + col], l);
        x = fmaf(f, o.x, x);
        y = fmaf(f, o.y, y);
    }
    dec_write2(p, join.x, h.first + col, dim, x / l, y / l);
    if (dim == 0) dec_write_lse(p, join.x, h.first + col, m, l);
}

// Launches for one format; `ctas` CTAs. Returns the kernels launched.
void launch_decode_f32(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int ctas);
void launch_decode_f16(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int ctas);
void launch_decode_q8_0(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int ctas);
void launch_decode_f8(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int ctas);

template <int FMT, int HD, int NT, bool WIDE> void launch_decode_as(cudaStream_t s, const DecodeParams & p, int ctas) {
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    auto kern = attention_decode_kernel<FMT, HD, NT, WIDE>;
    YK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::LAYOUT_BYTES));
    launch_k(kern, (unsigned)ctas, S::W * 32, S::LAYOUT_BYTES, s, p);
    launch_k(attention_decode_join_kernel<HD, S::COLS>, dim3((unsigned)ctas, S::COLS), HD / 2, 0, s, p);
}
template <int FMT, int HD, int NT> void launch_decode_tiles(cudaStream_t s, const DecodeParams & p, int ctas) {
    if (p.dtype == YUUKA_DTYPE_F32) launch_decode_as<FMT, HD, NT, true>(s, p, ctas);
    else launch_decode_as<FMT, HD, NT, false>(s, p, ctas);
}
template <int FMT, int NT> void launch_decode_dims(cudaStream_t s, const DecodeParams & p, int head_dim, int ctas) {
    if (head_dim == 64) launch_decode_tiles<FMT, 64, NT>(s, p, ctas);
    else if (head_dim == 128) launch_decode_tiles<FMT, 128, NT>(s, p, ctas);
    else launch_decode_tiles<FMT, 256, NT>(s, p, ctas);
}

}  // namespace yk
