// Attention of one new token per sequence over a paged cache (yuuka_attention_decode): the kernel.
//
// Mathematics. A unit is one KV head of one row of the batch, with up to 8 NT of the query heads that share it as columns.
// Its keys are taken 16 or 32 at a time: S^T = K Q^T (keys as the rows of the product, heads as its 8-wide columns), running
// maximum m and sum l per head, O^T += V^T P^T. Scores live in the base-2 domain, s = (scale log2 e) q.k, and probabilities
// carry a factor of 2^11 (over F32 pools none), p = 2^(s - m + 11). m is the maximum when the sums were last rescaled, which they are only when a score
// passes it by 2^4 (in the first tiles, mostly), so the largest p is 2^15, those down to 2^-25 of 2^m stay normal in f16, and
// what is rounded away is below 2^-36 of it. (A slack of 2^8 with a factor of 2^7 took as long.)
//
// What bounds it: the bytes of the cache, read once, over F32 and F16 pools (77 to 100 % of the memory's measured 6.54 TB/s
// for long sequences; F32 with heads of 256 or many columns, whose products are three to one, 41 to 78). Over Q8_0 (30 to 54 %) and F8 (41 to
// 75 %) the chain of instructions from a tile's bytes to its products takes longer than the bytes' way (28 and 40 % of the issue
// slots, with the two to four warps a scheduler that registers allow). The products run on mma.sync, whose operands a warp
// brings from shared memory into the fragments it needs: with one to eight query heads to a KV head the large tensor-core
// tiles would be empty but for a few columns, and the narrow ones take 10 to 40 % of the issue rate. The dimension that a
// product sums over may be taken in any order and a fragment's rows may stand for any dimensions, so a lane reads 16 bytes
// that lie side by side and takes them as its part of four products' operands; of V it reads the same dimensions of four keys,
// whose halves byte permutations pair up.
//
// A warp has a ring of tiles of its own in shared memory, K and V in turn, that cp.async fills several tiles ahead: no barrier of
// the CTA is waited for. Copies go by lines of 128 bytes.
//
// Work is cut at the granularity of warps. A team of as many warps as a row has units (KV heads) takes a run of tiles, each
// warp one head of the same keys, so that the heads of a token, which lie side by side in the pool, are read at about the same
// time. The rows' tiles form one sequence that the teams share evenly, wherever a run begins and ends, with its copies running
// ahead across rows. So batches of any mixture of lengths load the machine evenly, and the grid does not depend on the lengths,
// which only the device knows. A run that ends inside a row leaves a partial (O, m, l) in scratch memory, and a second kernel
// joins those of a row, always in the order of the keys, so results do not depend on timing.
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
    int warps;         // of the grid
    float * partial;   // [teams][units][2][part floats]: what a run leaves of its first row (0) and of its last one (1); sums l with a sign: to be done again
    int4 * joins;      // [2][DEC_WARPS] units that several teams share, few and many: x row, y unit of the row, z first and w last team
    int2 * far;        // [DEC_FAR_MOST] runs that have whole rows to be done again: x unit, y team
    int * counters;    // zero between calls: joins of both lists, runs in far, CTAs of the joining kernel done
};

constexpr int DEC_WARPS = 4096;         // of a grid, at most
constexpr size_t DEC_PARTIAL_BYTES = 40u << 20;  // two of the 1184 warps with the largest sums (16 columns of 256) take 39
enum { DEC_SHORT, DEC_LONG, DEC_FAR, DEC_DONE, DEC_COUNTERS };
constexpr int DEC_SHORT_MOST = 32;      // partials that a warp joins
constexpr int DEC_FAR_MOST = 16384;     // runs to do again: of each warp one, or of each unit where those are more (65536 / 8 + 1024 at most)
constexpr float DEC_LOWEST = -3.0e38f;  // of running maxima: finite, so that a score of -infinity weighs nothing even in a run without others
constexpr float DEC_SLACK = 4.0f;       // log2 of what a score may pass the running maximum by before sums are rescaled
constexpr int DEC_SMEM_SM = 233472;     // shared memory of an SM

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
template <int BYTES> __device__ __forceinline__ void dec_copy(uint32_t dst, const uint8_t * src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// 16 bytes, of which n are read and the others become zeros
__device__ __forceinline__ void dec_copy_part(uint32_t dst, const uint8_t * src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// What the tensor core's tf32 (an f32 cut off behind 10 bits of its fraction) leaves of an f32, as a tf32: rounded, since
// the cutting alone would make all scores 2^-22 too small.
__device__ __forceinline__ uint32_t dec_rest(uint32_t x) {
    return __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffffe000u)) + 0x1000u;
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
// four E4M3 as two pairs of f16
__device__ __forceinline__ uint2 dec_e4m3(uint32_t four) {
    uint2 h;
    asm volatile("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
                 : "=r"(h.x), "=r"(h.y)
                 : "r"(four));
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
// the products as two parts (22 bits); otherwise f16 or bf16 and one part (11 bits: as much as an f16 output has, and with its
// rounding an error of the square root of two of one).
template <int FMT, int HD, int NT, bool WIDE> struct DecodeShape {
    static constexpr bool IS_F32 = FMT == YUUKA_KV_F32, IS_Q8 = FMT == YUUKA_KV_Q8_0, IS_F8 = FMT == YUUKA_KV_F8;
    // Warps of a CTA and CTAs of an SM: twelve warps an SM, or eight where the sums, queries and copies of 256 dimensions take the
    // registers (at 12 and 8 instead of 8 and 4 warps, 8 sequences of 32768 with 8 KV heads of 128 took 160 us instead of 164, 32 of
    // 256 to 4000 with 4 of 256 took 41 instead of 44; 24 of 8000 in F8 with 16 query heads to each of 4 KV heads of 256 took 110 with
    // eight, 145 with four). Sixteen with heads of 64 and 16-bit queries (24 of 8000 with 16 KV heads of 64: Q8_0 140 instead of 152,
    // F8 126 instead of 133, F16 125 instead of 130; with heads of 128 they spill: F8 109 instead of 90). With f32 queries F8 does
    // better with eight there (118 instead of 133; Q8_0 181 instead of 159, F16 the same). Four where eight spill what a tile needs.
    // Small CTAs are resident sooner: one short sequence took 7.4 us with 2 of four warps, 7.6 with one of eight.
    static constexpr bool NARROW = NT == 2 || (IS_F32 && HD > 64) || (WIDE && (HD == 128 || (IS_F8 && HD == 64)));
    static constexpr int W = 4, RESIDENT = HD == 256 ? (IS_F32 || (FMT == YUUKA_KV_F16 && NT == 2 && WIDE) ? 1 : 2)
                                                     : (NARROW ? 2 : HD == 64 && !WIDE && !IS_F32 ? 4 : 3);
    // keys of a tile: sixteen make one row tile of the products, and two of them share the walk, the maximum and the queries' reads
    // where registers allow (64 sequences of 500 to 8000 in F8: 106 -> 99 us). With f32 queries and heads of 128 eight warps of two
    // beat twelve of one: 24 of 8000 with 8 KV heads 124 instead of 142 us (F16), 101 instead of 127 (F8), 142 instead of 156 (Q8_0).
    static constexpr int HALVES = HD == 256 || (HD == 128 && (IS_F32 || (WIDE && NT == 2))) ? 1 : 2, KEYS = 16 * HALVES;
    static constexpr int COLS = 8 * NT, PARTS = WIDE ? 2 : 1;
    // log2 of the factor that probabilities carry into f16 (tf32 has the exponents of f32, and sums of large values room without one)
    static constexpr float P_LOG2 = IS_F32 ? 0.0f : 11.0f;
    // Q8_0, F8: ratio (log2) of the scales of V from which on a row is done again, in f32. Probabilities of 2^11 for the heaviest key enter
    // the products in units of the largest scale, rounded to half of f16's 2^-24: at this ratio a key of the smallest scale that has all
    // the weight is held to 2^-36 * 2 * 2^10 = 2^-25 (f32 queries), or 2^-21, of itself.
    static constexpr int FAR_LOG2 = WIDE ? 10 : 14;
    // Q8_0: a head's blocks of 34 bytes, copied as the 16-byte pieces that hold them, which begin up to 12 bytes before. (Copied by
    // words, 24 sequences of 8000 with 16 KV heads of 64 took 176 us.) A piece more or less from key to key would put the lanes'
    // reads of V on the same banks.
    static constexpr int Q8_PIECES = HD == 64 ? 5 : (HD == 128 ? 9 : 17), Q8_ROW = 16 * Q8_PIECES;
    static constexpr bool Q8_STARTS = IS_Q8 && HD != 256;  // a head of 256 is 17 pieces itself
    // F8: a lane's piece of V, 16 dimensions of 128 or 8 of 64; the scales of the tile's K and V lie behind K
    static constexpr int F8_V = HD == 64 ? 8 : 16;
    static constexpr int K16 = IS_F32 ? HD * 64 : (IS_Q8 ? 16 * Q8_ROW : (IS_F8 ? HD * 16 : HD * 32));  // bytes of sixteen keys
    static constexpr int V16 = IS_F32 ? HD * 64 : (IS_Q8 ? 16 * Q8_ROW : (IS_F8 ? HD * 16 : HD * 32));
    // (behind the tile: F8's scales of K and V; where in their first pieces Q8_0's rows begin)
    static constexpr int K_BYTES = K16 * HALVES + (IS_F8 ? 8 * KEYS : Q8_STARTS ? 4 * KEYS : 0), V_BYTES = V16 * HALVES + (Q8_STARTS ? 4 * KEYS : 0);
    // Rows of the other formats, K and V: their 16-byte pieces are copied by lines of 128 bytes, eight neighbouring lanes to a
    // line. (With lanes that copy what they will read themselves, four to a piece of K and every fourth to a line of V, the SMs
    // fetched V's sectors twice: 1.61 GB for 1.07.) Pieces trade places within their line so that the eight lanes of a read find
    // them on different banks: four pieces of two keys (K), two pieces of every other of eight keys (V).
    static constexpr int ROW = IS_Q8 ? 0 : IS_F32 ? HD * 4 : IS_F8 ? HD : HD * 2;
    static constexpr int LINE = ROW >= 128 ? 128 : 64, LANES = LINE / 16;  // bytes and lanes of a line
    // where piece q of a key's row lies
    __device__ static __forceinline__ uint32_t k_piece(int key, int q) { return key * ROW + 16 * (LINE == 128 ? q ^ ((key & 1) << 2) : q); }
    __device__ static __forceinline__ uint32_t v_piece(int key, int q) { return key * ROW + 16 * (q ^ ((key >> 1 & (LINE == 128 ? 3 : 1)) << 1)); }
    static constexpr int SLOT = (K_BYTES > V_BYTES ? K_BYTES : V_BYTES);
    static constexpr int PART_FLOATS = COLS * (HD + 2);
    // queries in registers, or in shared memory where the sums leave too few (f32: 8 heads of all dimensions, split at use)
    static constexpr bool Q_SHARED = IS_F32 || HD / 4 * NT + HD / 8 * PARTS * NT > 128;
    static constexpr int Q_BYTES = !Q_SHARED ? 0 : (IS_F32 ? 8 * HD * 4 : COLS * HD * 2 * PARTS);
    static constexpr int WARP_BYTES = (DEC_SMEM_SM / RESIDENT - 1536) / W / 16 * 16;  // (the rest: what the system keeps of a CTA's share)
    static constexpr int FIT = (WARP_BYTES - Q_BYTES) / SLOT;
    static constexpr int SLOTS = FIT > 8 ? 8 : FIT;  // K and V of a tile take one each
    static constexpr int AHEAD = SLOTS - 1;
    static constexpr int RING = SLOTS * SLOT;
    static_assert(SLOTS >= 2, "a warp's shared memory");
    static constexpr int LAYOUT_BYTES = W * (RING + Q_BYTES);
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
            return blk * 32 + ((blk & 1) ? 4 * (t + 4 * h) + 2 * half : (4 * (1 + t + 4 * h) - 2 + 2 * half) & 31);
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
__host__ __device__ __forceinline__ DecodeSpan decode_span(const DecodeParams & p, int b, int keys, int & bad) {  // keys of a tile
    DecodeSpan s;
    const int n = kv_load(p.lens + b);
    s.seq = p.seq_ids ? kv_load(p.seq_ids + b) : b;
    bad = 0;
    if ((unsigned)s.seq >= (unsigned)p.cache.sequences) bad = KV_BAD_SEQUENCE;
    else if (n < 0 || n > p.cache.capacity) bad = KV_BAD_POSITION;
    s.end = bad ? 0 : n;
    s.first = p.window > 0 && s.end > p.window ? s.end - p.window : 0;
    s.tiles = s.end > s.first ? (s.end - s.first - 1) / keys + 1 : 1;
    if (bad) s.seq = -1;
    return s;
}
__device__ __forceinline__ DecodeSpan decode_span(const DecodeParams & p, int b, int keys) {
    int bad;
    return decode_span(p, b, keys, bad);
}

// A place in the sequence of tiles: the next one of row b.
template <int KEYS> struct DecodeCursor {
    int b;
    int pos, end;           // its first key; behind the row's last key
    int left;               // tiles of the row from here on
    int first, tiles, seq;  // of the row
    __device__ __forceinline__ void row(const DecodeParams & p) {
        const DecodeSpan s = decode_span(p, b, KEYS);
        first = s.first;
        end = s.end;
        tiles = s.tiles;
        seq = s.seq;
    }
    // the whole warp: tile `begin` of the sequence (less than its length: some row holds it)
    __device__ __forceinline__ void seek(const DecodeParams & p, unsigned begin) {
        const int lane = threadIdx.x & 31;
        unsigned before = 0;
        b = 0;
        for (int base = 0; base < p.batch; base += 32) {
            const int at = base + lane;
            const unsigned mine = at < p.batch ? (unsigned)decode_span(p, at, KEYS).tiles : 0;
            unsigned sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + sum > begin);
            if (hit) {
                const int first_hit = __ffs(hit) - 1;
                b = base + first_hit;
                before += __shfl_sync(0xffffffffu, sum - mine, first_hit);
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        row(p);
        const int tile = min((int)(begin - before), tiles - 1);  // (it is less, unless lengths change under the call)
        pos = first + tile * KEYS;
        left = tiles - tile;
    }
    __device__ __forceinline__ void next(const DecodeParams & p) {
        pos += KEYS;
        if (--left > 0) return;
        if (++b < p.batch) row(p);
        pos = first;
        left = tiles;
    }
};

// ---- results -------------------------------------------------------------------------------------------------------

// N neighbouring values (2, or a multiple of 4) as words, through the read-only path: loads may be moved over stores, and no
// branch on the type stands between them.
template <bool WIDE, int N> struct DecodeRaw {
    static constexpr int WORDS = WIDE ? N : N / 2;
    uint32_t w[WORDS];
    __device__ __forceinline__ void fetch(const float * from) {  // scratch memory: not through the read-only path
        static_assert(WIDE, "f32");
#pragma unroll
        for (int i = 0; i < WORDS; i += N == 2 ? 2 : 4) {
            if constexpr (N == 2) *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(from);
            else *reinterpret_cast<uint4 *>(w + i) = *reinterpret_cast<const uint4 *>(from + i);
        }
    }
    __device__ __forceinline__ void load(const void * base, int64_t at) {
        const uint32_t * src = reinterpret_cast<const uint32_t *>(base) + (WIDE ? at : at / 2);
        if constexpr (WORDS == 1) w[0] = __ldg(src);
        else if constexpr (WORDS == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(src));
            w[0] = v.x;
            w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src + i));
                w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ float2 pair(int i, int dtype) const {  // values 2 i and 2 i + 1
        if constexpr (WIDE) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else {
            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(w + i));
            const float2 b = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            return dtype == YUUKA_DTYPE_F16 ? h : b;
        }
    }
    __device__ __forceinline__ void set(float2 x, int dtype) {  // values 0 and 1 (which the type can hold)
        if constexpr (WIDE) {
            w[0] = __float_as_uint(x.x);
            w[1] = __float_as_uint(x.y);
        } else if (dtype == YUUKA_DTYPE_F16) {
            w[0] = dec_pack(x.x, x.y);
        } else {
            w[0] = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
        }
    }
};
// the gates of N neighbouring values of a head: what the values are multiplied with
template <bool WIDE, int N> __device__ __forceinline__ void dec_gates(const DecodeParams & p, const DecodeRaw<WIDE, N> & raw, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const float2 z = raw.pair(i, p.dtype);
        if constexpr (WIDE) {
            // of e^-|z|, which does not overflow: within 2^-22 of the gate. (The approximate exponential's error grows with |z|.)
            const float ex = expf(-fabsf(z.x)), ey = expf(-fabsf(z.y));
            f[2 * i] = (z.x < 0.0f ? ex : 1.0f) / (1.0f + ex);
            f[2 * i + 1] = (z.y < 0.0f ? ey : 1.0f) / (1.0f + ey);
        } else {
            // (approximate exponential and reciprocal: (4 + |z|) 2^-23, for outputs that are rounded to 2^-11 or 2^-8)
            f[2 * i] = __fdividef(1.0f, 1.0f + __expf(-z.x));
            f[2 * i + 1] = __fdividef(1.0f, 1.0f + __expf(-z.y));
        }
    }
}
// N neighbouring values of a head's result, rounded to the output's type
template <bool WIDE, int N> __device__ __forceinline__ void dec_write(const DecodeParams & p, int b, int head, int dim, const float (&x)[N]) {
    const int64_t at = b * p.out_row + head * p.out_head + dim;
    if constexpr (WIDE) {
        float * dst = reinterpret_cast<float *>(p.out) + at;
        if constexpr (N == 2) *reinterpret_cast<float2 *>(dst) = make_float2(x[0], x[1]);
        else
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        return;
    }
    uint32_t raw[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        if (p.dtype == YUUKA_DTYPE_F16) *reinterpret_cast<__half2 *>(raw + i) = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        else *reinterpret_cast<__nv_bfloat162 *>(raw + i) = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    }
    uint16_t * dst = reinterpret_cast<uint16_t *>(p.out) + at;
    if constexpr (N == 2) *reinterpret_cast<uint32_t *>(dst) = raw[0];
    else if constexpr (N == 4) *reinterpret_cast<uint2 *>(dst) = make_uint2(raw[0], raw[1]);
    else
#pragma unroll
        for (int i = 0; i < N / 2; i += 4) *reinterpret_cast<uint4 *>(dst + 2 * i) = make_uint4(raw[i], raw[i + 1], raw[i + 2], raw[i + 3]);
}
__device__ __forceinline__ void dec_write_lse(const DecodeParams & p, int b, int head, float m, float l) {
    if (p.lse) p.lse[(int64_t)b * p.heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
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

// Whether a join is one that this call's teams can have left. (Calls that share scratch memory against the rule may read one
// another's joins: wrong results, but no memory beyond the partial sums that this call's own warps have.)
__host__ __device__ __forceinline__ bool decode_join_sound(const DecodeParams & p, const int4 & j) {
    const int units = p.cache.kv_heads * p.head_tiles;
    return (unsigned)j.x < (unsigned)p.batch && (unsigned)j.y < (unsigned)units && j.z >= 0 && j.z < j.w && j.w < p.warps / units;
}

// ---- the kernel ----------------------------------------------------------------------------------------------------

template <int FMT, int HD, int NT, bool WIDE>
__global__ void __launch_bounds__(DecodeShape<FMT, HD, NT, WIDE>::W * 32, DecodeShape<FMT, HD, NT, WIDE>::RESIDENT) attention_decode_kernel(const DecodeParams p) {
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    constexpr int W = S::W, COLS = S::COLS, AHEAD = S::AHEAD, CHUNKS = S::CHUNKS, DPL = S::DPL, HALVES = S::HALVES, KEYS = S::KEYS;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * S::RING);
    const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(smem + W * S::RING + warp * S::Q_BYTES) + lane * 16;
    pdl_entry();

    // this warp's unit and its team's run of tiles
    unsigned total = 0;  // (below 2^31: the host has checked)
    for (int b = lane; b < p.batch; b += 32) {
        int bad;
        total += decode_span(p, b, KEYS, bad).tiles;
        if (bad && p.status && blockIdx.x == 0 && warp == 0) atomicOr(p.status, bad);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    const unsigned units = p.cache.kv_heads * p.head_tiles, warps = gridDim.x * W, self = blockIdx.x * W + warp;
    const unsigned teams = max(warps / units, 1u), team = min(self / units, units > warps ? 0u : ~0u);
    const unsigned share = (total + teams - 1) / teams;
    const unsigned begin = team * share;
    const int count = team < teams && begin < total ? (int)min(share, total - begin) : 0;
#pragma unroll 1
    for (unsigned unit = units > warps ? self : self - team * units; unit < units; unit += warps) {
        if (count == 0) break;
        DecodeCursor<KEYS> use;
        use.seek(p, begin);

        // -- copies. Keys behind the last one of a unit's last tile repeat it (their probabilities become zero), so a copy is
        // always whole; a tile of a bad block becomes NaN, and a unit without keys copies nothing.
        DecodeCursor<KEYS> ahead = use;
        int fetched = 0;                   // tiles of the run whose V has been asked for
        unsigned block_of = 0, within = 0; // of key lane % KEYS of the next tile
        unsigned pool_row = 0;
        bool copies = false;
        // the pools at the unit's head and this lane's piece
        constexpr int HEAD_BYTES = FMT == YUUKA_KV_F32 ? HD * 4 : (FMT == YUUKA_KV_F16 ? HD * 2 : (FMT == YUUKA_KV_Q8_0 ? HD / 32 * 34 : HD));
        const int kv_head = unit / p.head_tiles;
        const unsigned head_at = kv_head * HEAD_BYTES;
        [[maybe_unused]] const uint8_t * const k_at = p.cache.k + head_at + 16 * (lane & (S::LANES - 1));
        [[maybe_unused]] const uint8_t * const v_at = p.cache.v + head_at + 16 * (lane & (S::LANES - 1));
        [[maybe_unused]] const uint64_t pool_bytes = (uint64_t)p.cache.pool_blocks * p.cache.block_size * (uint64_t)p.cache.row_bytes;
        const int32_t * table = nullptr;
        const unsigned row_bytes = (unsigned)p.cache.row_bytes;
        auto look_up = [&] {
            if (ahead.pos >= ahead.end) return;
            const int pos = min(ahead.pos + (lane & (KEYS - 1)), ahead.end - 1);
            const int page = p.cache.shift >= 0 ? pos >> p.cache.shift : pos / p.cache.block_size;
            within = pos - page * p.cache.block_size;
            block_of = (unsigned)__ldg(table + page);
        };
        auto enter = [&] {  // the row that `ahead` has come to
            table = p.cache.tables + (int64_t)max(ahead.seq, 0) * p.cache.table_stride;
        };
        enter();
        look_up();
        uint32_t put = ring;  // slot that is filled next
        auto fetch = [&](auto is_v) {
            constexpr bool V = decltype(is_v)::value;
            if (fetched < count) {
                if constexpr (!V) {
                    copies = false;
                    if (ahead.pos < ahead.end) {
                        copies = !__any_sync(0xffffffffu, block_of >= (unsigned)p.cache.pool_blocks);
                        pool_row = block_of * (unsigned)p.cache.block_size + within;
                        if (!copies) {
                            if (lane == 0 && p.status) atomicOr(p.status, KV_BAD_BLOCK);
                            for (uint32_t at = put + 16 * lane; at < put + S::SLOT; at += 512) dec_sts4(at, make_uint4(~0u, ~0u, ~0u, ~0u));
                        }
                    }
                }
                if constexpr (S::Q8_STARTS) {  // written for tiles that copy nothing as well: they are read all the same
                    __syncwarp();
                    if (lane < KEYS) dec_sts(put + S::K16 * HALVES + 4 * lane, copies ? (uint32_t)((uint64_t)pool_row * row_bytes + head_at) & 15u : 0u);
                }
                if (copies) {
                    [[maybe_unused]] auto row_of = [&](int key) { return (V ? v_at : k_at) + (uint64_t)__shfl_sync(0xffffffffu, pool_row, key) * row_bytes; };
                    if constexpr (S::IS_Q8) {
                        const uint8_t * const base = V ? p.cache.v : p.cache.k;
#pragma unroll
                        for (int i = 0; i < (KEYS * S::Q8_PIECES + 31) / 32; i++) {
                            const int at = 32 * i + lane, key = at / S::Q8_PIECES, piece = at - key * S::Q8_PIECES;
                            const uint64_t from = (((uint64_t)__shfl_sync(0xffffffffu, pool_row, key & 31) * row_bytes + head_at) & ~15ull) + 16 * piece;
                            // (the last piece of the pool's last row may reach beyond the pool)
                            if (32 * i + 31 < KEYS * S::Q8_PIECES || key < KEYS)
                                dec_copy_part(put + key * S::Q8_ROW + 16 * piece, base + from, (int)min((uint64_t)16, pool_bytes - min(from, pool_bytes)));
                        }
                    } else {
                        constexpr int AT_ONCE = 32 / S::LANES;  // keys
#pragma unroll
                        for (int k = 0; k < KEYS / AT_ONCE; k++) {
                            const int key = AT_ONCE * k + lane / S::LANES, q = lane & (S::LANES - 1);
                            const uint8_t * src = row_of(key);
                            const uint32_t dst = put + (V ? S::v_piece(key, q) : S::k_piece(key, q));
#pragma unroll
                            for (int i = 0; i < S::ROW / S::LINE; i++) dec_copy<16>(dst + S::LINE * i, src + S::LINE * i);
                        }
                        if constexpr (FMT == YUUKA_KV_F8 && !V) {
                            // scales of K and behind them of V
                            const uint64_t at = (uint64_t)pool_row * row_bytes + (p.cache.kv_heads * HD + 4 * kv_head);
                            const uint32_t dst = put + S::K16 * HALVES + 4 * lane;
                            if constexpr (HALVES == 2) {
                                dec_copy<4>(dst, p.cache.k + at);
                                dec_copy<4>(dst + 128, p.cache.v + at);
                            } else {
                                dec_copy<4>(dst, (lane < 16 ? p.cache.k : p.cache.v) + at);
                            }
                        }
                    }
                }
                if constexpr (V) {
                    if (++fetched < count) {
                        const bool other = ahead.left == 1;
                        ahead.next(p);
                        if (other) enter();
                        look_up();
                    }
                }
            }
            put = put + S::SLOT == ring + S::RING ? ring : put + S::SLOT;
            dec_commit();
        };
#pragma unroll 1
        for (int i = 0; i < AHEAD / 2; i++) {
            fetch(std::false_type());
            fetch(std::true_type());
        }
        if constexpr (AHEAD & 1) fetch(std::false_type());

        // -- per unit: queries, statistics and sums
        constexpr int QM = HD / 16;  // 16-bit products over the head dimension
        uint32_t q[S::Q_SHARED ? 1 : NT][S::Q_SHARED ? 1 : S::PARTS][S::Q_SHARED ? 1 : QM][2];
        float scale[NT][2];          // of the columns' scores, not negative: a negative scale's sign goes into the queries
        float m[NT][2], l[NT][2];    // l: of this lane's keys
        float o[NT][CHUNKS][DPL / 2][4];
        float v_scale = 1.0f;        // Q8_0, F8: o is in units of it (a power of two)
        [[maybe_unused]] bool again = false;      // the run has whole rows for the second kernel to do again
        [[maybe_unused]] uint32_t v_least = ~0u;  // smallest scale of V but zero that the lane has seen: bits of its magnitude less one (Q8_0: f16)
        bool from_start = false, fresh = true;

        auto load_queries = [&] {
            const DecodeHeads h = decode_heads(p, unit);
            const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int col = nt * 8 + g;
                const bool has = col < h.count;
                const int64_t at = use.b * p.q_row + (h.first + (has ? col : 0)) * p.q_head;
                if constexpr (S::IS_F32) {
                    // dimensions 16 i + 4 t .. + 3 of head g
                    DecodeRaw<WIDE, 4> raw[HD / 16];
#pragma unroll
                    for (int i = 0; i < HD / 16; i++) raw[i].load(p.q, at + 16 * i + 4 * t);
                    const float f = has ? sign : 0.0f;
#pragma unroll
                    for (int i = 0; i < HD / 16; i++) {
                        const float2 x = raw[i].pair(0, p.dtype), y = raw[i].pair(1, p.dtype);
                        dec_sts4(q_at + 512 * i, make_uint4(__float_as_uint(x.x * f), __float_as_uint(x.y * f), __float_as_uint(y.x * f), __float_as_uint(y.y * f)));
                    }
                    scale[nt][0] = scale[nt][1] = fmaxf(fabsf(p.scale_log2), 1e-37f);
                } else {
                    // scaled to a largest magnitude of 2^14 .. 2^15, so that two f16 parts hold 22 bits of what matters
                    DecodeRaw<WIDE, 2> raw[2 * QM];
#pragma unroll
                    for (int i = 0; i < 2 * QM; i++) raw[i].load(p.q, at + S::q_dim(i >> 1, i & 1, t));
                    float amax = 0.0f;
                    [[maybe_unused]] float least = INFINITY;
#pragma unroll
                    for (int i = 0; i < 2 * QM; i++) {
                        const float2 x = raw[i].pair(0, p.dtype);
                        amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
                        if constexpr (FMT == YUUKA_KV_F16) least = fminf(least, fminf(fabsf(x.x), fabsf(x.y)));
                    }
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    const int e = min(max((int)(__float_as_uint(amax) >> 23), 15), 254);
                    if constexpr (FMT == YUUKA_KV_F16) {
                        // no first part is zero but of a zero: its sign decides over an infinite key. 2^-24 in its units, 2^-38 of the largest
                        // (beside an infinite query nothing else counts)
                        const float low = e > 38 && e < 254 ? __int_as_float((e - 38) << 23) : 0.0f;
                        if (least < low)
#pragma unroll
                            for (int i = 0; i < 2 * QM; i++) {
                                float2 x = raw[i].pair(0, p.dtype);
                                if (x.x != 0.0f) x.x = copysignf(fmaxf(fabsf(x.x), low), x.x);
                                if (x.y != 0.0f) x.y = copysignf(fmaxf(fabsf(x.y), low), x.y);
                                raw[i].set(x, p.dtype);
                            }
                    }
                    const float up = has ? sign * __int_as_float((268 - e) << 23) : 0.0f;                          // 2^(14 - (e - 127))
                    const float down = fmaxf(fabsf(p.scale_log2) * __int_as_float((e - 14) << 23), 1e-37f);        // |scale| / up
                    scale[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
                    scale[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
                    for (int i = 0; i < QM; i++) {
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            float2 x = raw[2 * i + half].pair(0, p.dtype);
                            x.x *= up;
                            x.y *= up;
                            hi[half] = dec_pack(x.x, x.y);
                            const float2 r = dec_unpack(hi[half]);
                            if constexpr (S::IS_Q8 || S::IS_F8)  // (of an infinite query not NaN: its first part is to decide)
                                lo[half] = dec_pack(fmaxf(x.x - r.x, -65504.0f), fmaxf(x.y - r.y, -65504.0f));
                            else lo[half] = dec_pack(x.x - r.x, x.y - r.y);
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
            return v_scale < 1.7e38f ? __uint_as_float(0x7f000000u - __float_as_uint(v_scale)) : 1.0f / v_scale;  // (a power of two)
        };
        // o += a P^T for product j of a chunk. The tensor core cuts sums off instead of rounding them: over thousands of tiles
        // that would cost an f32 result 2^-17, so such a tile is summed on its own and added in f32
        auto add_values = [&](float (&acc)[4], int nt, const uint32_t (&a)[HALVES][4], const uint32_t (&b)[HALVES][NT][S::PARTS][2]) {
            if constexpr (WIDE) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < HALVES; h++) dec_mma16(d, a[h][0], a[h][1], a[h][2], a[h][3], b[h][nt][S::PARTS - 1][0], b[h][nt][S::PARTS - 1][1]);
#pragma unroll
                for (int h = 0; h < HALVES; h++) dec_mma16(d, a[h][0], a[h][1], a[h][2], a[h][3], b[h][nt][0][0], b[h][nt][0][1]);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[e] += d[e];
            } else {
#pragma unroll
                for (int h = 0; h < HALVES; h++) dec_mma16(acc, a[h][0], a[h][1], a[h][2], a[h][3], b[h][nt][0][0], b[h][nt][0][1]);
            }
        };

        uint32_t take = ring;  // slot that is used next
#pragma unroll 1
        for (int it = 0; it < count; it++) {
            // ---- K: scores
            dec_wait<AHEAD - 1>();
            __syncwarp();  // (lanes read what others have copied, and copy over what others have read)
            if constexpr (AHEAD & 1) fetch(std::true_type());
            else fetch(std::false_type());
            const uint32_t ks = take;
            take = take + S::SLOT == ring + S::RING ? ring : take + S::SLOT;

            if (fresh) {
                fresh = false;
                from_start = use.left == use.tiles;
                load_queries();
                v_scale = __uint_as_float(0x00800000u);
                v_least = ~0u;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    m[nt][0] = m[nt][1] = DEC_LOWEST;
                    // (a row that is out of range has no keys and becomes NaN)
                    l[nt][0] = l[nt][1] = use.seq < 0 ? __uint_as_float(0x7fffffffu) : 0.0f;
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                        for (int j = 0; j < DPL / 2; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[nt][c][j][e] = 0.0f;
                }
            }
            const int keys = use.end - use.pos;  // of the unit from here on; 0 for a row without any

            // probabilities as fragments: keys become the dimension that is summed over
            uint32_t pb[HALVES][NT][S::PARTS][2];
            float sh[HALVES][NT][4];
            auto fragments = [&](int h, float f0, float f1) {  // of the h-th sixteen keys, with factors of keys g and g + 8
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float x0 = sh[h][nt][0] * f0, x1 = sh[h][nt][1] * f0, y0 = sh[h][nt][2] * f1, y1 = sh[h][nt][3] * f1;
                    const uint32_t hx = dec_pack(x0, x1), hy = dec_pack(y0, y1);
                    pb[h][nt][0][0] = dec_transpose(hx);
                    pb[h][nt][0][1] = dec_transpose(hy);
                    if constexpr (WIDE) {
                        const float2 rx = dec_unpack(hx), ry = dec_unpack(hy);
                        pb[h][nt][1][0] = dec_transpose(dec_pack(x0 - rx.x, x1 - rx.y));
                        pb[h][nt][1][1] = dec_transpose(dec_pack(y0 - ry.x, y1 - ry.y));
                    }
                }
            };
            if (keys > 0) {  // (uniform)
                float vd[HALVES][2];  // F8: scales of V of keys g and g + 8
#pragma unroll
                for (int half = 0; half < HALVES; half++) {
                float (&s)[NT][4] = sh[half];
                const uint32_t kh = ks + half * S::K16;
                float s2[NT][4];
                [[maybe_unused]] float s3[NT][4] = {};
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[nt][e] = s2[nt][e] = 0.0f;
                if constexpr (S::IS_F32) {
                    // three products of tf32 parts: hi hi, hi lo, lo hi (the tensor core itself drops what a first part leaves). What
                    // the first ones cut off counts (see add_values): two at a time, added in f32
#pragma unroll
                    for (int c = 0; c < HD / 16; c++) {
                        const uint4 ka = dec_lds4(kh + S::k_piece(g, 4 * c + t)), kb = dec_lds4(kh + S::k_piece(g + 8, 4 * c + t));
                        const uint4 f = dec_lds4(q_at + 512 * c);
                        const uint32_t a[8] = {ka.x, kb.x, ka.y, kb.y, ka.z, kb.z, ka.w, kb.w};
                        const uint32_t b[4] = {f.x, f.y, f.z, f.w};
                        uint32_t al[8], bl[4];
#pragma unroll
                        for (int i = 0; i < 8; i++) al[i] = dec_rest(a[i]);
#pragma unroll
                        for (int i = 0; i < 4; i++) bl[i] = dec_rest(b[i]);
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        dec_mma8(d, a[0], a[1], a[2], a[3], b[0], b[1]);
                        dec_mma8(d, a[4], a[5], a[6], a[7], b[2], b[3]);
                        dec_mma8(s2[0], al[0], al[1], al[2], al[3], b[0], b[1]);
                        dec_mma8(s2[0], al[4], al[5], al[6], al[7], b[2], b[3]);
                        if constexpr (WIDE) {  // (16-bit queries have no second part)
                            dec_mma8(s2[0], a[0], a[1], a[2], a[3], bl[0], bl[1]);
                            dec_mma8(s2[0], a[4], a[5], a[6], a[7], bl[2], bl[3]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) s[0][e] += d[e];
                    }
                } else if constexpr (S::IS_Q8) {
                    // keys g and g + 8
                    uint32_t ka = kh + g * S::Q8_ROW, kb = ka + 8 * S::Q8_ROW;
                    if constexpr (S::Q8_STARTS) {
                        const uint32_t starts = ks + S::K16 * HALVES + 64 * half + 4 * g;
                        ka += dec_lds(starts);
                        kb += dec_lds(starts + 32);
                    }
#pragma unroll
                    for (int pair = 0; pair < HD / 64; pair++) {
                        uint32_t w[2][4];   // [key][word]: two of the even block, two of the odd one
                        float d[2][2];      // [key][block]
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint32_t at = (k ? kb : ka) + 68 * pair;
                            const uint2 even = make_uint2(dec_lds(at + 4 * (1 + t)), dec_lds(at + 4 * (5 + t)));
                            const uint2 odd = make_uint2(dec_lds(at + 4 * (9 + t)), dec_lds(at + 4 * (13 + t)));
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
                        for (int blk = 0; blk < 2; blk++) {
                            uint32_t a[2][4];
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t u0 = w[0][2 * blk + h], u1 = w[1][2 * blk + h];
                                a[h][0] = dec_int8<0>(u0);
                                a[h][1] = dec_int8<0>(u1);
                                a[h][2] = dec_int8<1>(u0);
                                a[h][3] = dec_int8<1>(u1);
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                for (int h = 0; h < 2; h++) {
                                    const uint4 f = query(nt, 4 * pair + 2 * blk + h);
                                    if constexpr (WIDE) dec_mma16(x, a[h][0], a[h][1], a[h][2], a[h][3], f.z, f.w);
                                    dec_mma16(x, a[h][0], a[h][1], a[h][2], a[h][3], f.x, f.y);
                                }
                                s[nt][0] = fmaf(x[0], d[0][blk], s[nt][0]);
                                s[nt][1] = fmaf(x[1], d[0][blk], s[nt][1]);
                                s[nt][2] = fmaf(x[2], d[1][blk], s[nt][2]);
                                s[nt][3] = fmaf(x[3], d[1][blk], s[nt][3]);
                            }
                        }
                    }
                } else if constexpr (S::IS_F8) {
#pragma unroll
                    for (int c = 0; c < HD / 64; c++) {
                        const uint4 ka = dec_lds4(kh + S::k_piece(g, 4 * c + t)), kb = dec_lds4(kh + S::k_piece(g + 8, 4 * c + t));
                        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint2 x = dec_e4m3(wa[i]), y = dec_e4m3(wb[i]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const uint4 f = query(nt, 4 * c + i);
                                dec_mma16((i & 1) ? s2[nt] : s[nt], x.x, y.x, x.y, y.y, f.x, f.y);
                                if constexpr (WIDE) dec_mma16((i & 1) ? s2[nt] : s[nt], x.x, y.x, x.y, y.y, f.z, f.w);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < HD / 32; c++) {
                        const uint4 ka = dec_lds4(kh + S::k_piece(g, 4 * c + t)), kb = dec_lds4(kh + S::k_piece(g + 8, 4 * c + t));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint4 f = query(nt, 2 * c), f2 = query(nt, 2 * c + 1);
                            dec_mma16(s[nt], ka.x, kb.x, ka.y, kb.y, f.x, f.y);
                            dec_mma16(s2[nt], ka.z, kb.z, ka.w, kb.w, f2.x, f2.y);
                            if constexpr (WIDE) {  // second parts on their own: their signs are any
                                dec_mma16(s3[nt], ka.x, kb.x, ka.y, kb.y, f.z, f.w);
                                dec_mma16(s3[nt], ka.z, kb.z, ka.w, kb.w, f2.z, f2.w);
                            }
                        }
                    }
                }
                // an infinity of K makes the sum of the first parts infinite or NaN as it should be, and nothing of the second parts,
                // which it meets with either sign or a zero
                if constexpr (!S::IS_Q8)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (!S::IS_F32 || fabsf(s[nt][e]) < INFINITY) s[nt][e] += s2[nt][e];
                            if constexpr (FMT == YUUKA_KV_F16 && WIDE)
                                if (fabsf(s[nt][e]) < INFINITY) s[nt][e] += s3[nt][e];
                        }
                if constexpr (S::IS_F8) {
                    const uint32_t at = ks + S::K16 * HALVES + 64 * half + 4 * g;
                    const float d0 = __uint_as_float(dec_lds(at)), d1 = __uint_as_float(dec_lds(at + 32));
                    vd[half][0] = __uint_as_float(dec_lds(at + 4 * KEYS));
                    vd[half][1] = __uint_as_float(dec_lds(at + 4 * KEYS + 32));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        s[nt][0] *= d0;
                        s[nt][1] *= d0;
                        s[nt][2] *= d1;
                        s[nt][3] *= d1;
                    }
                }
                }

                // ---- running maximum and sum; s becomes the probabilities of keys g (0, 1) and g + 8 (2, 3), columns 2t and 2t + 1
                if (keys < KEYS) {
#pragma unroll
                    for (int h = 0; h < HALVES; h++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (16 * h + g + 8 * (e >> 1) >= keys) sh[h][nt][e] = -INFINITY;
                }
                float top[NT][2];
                bool moved = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float mx = fmaxf(sh[0][nt][c], sh[0][nt][c + 2]);
                        if constexpr (HALVES == 2) mx = fmaxf(mx, fmaxf(sh[1][nt][c], sh[1][nt][c + 2]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        top[nt][c] = fmaxf(m[nt][c], mx * scale[nt][c]);
                        moved |= top[nt][c] > m[nt][c] + DEC_SLACK;
                    }
                if (__any_sync(0xffffffffu, moved)) {
                    float corr[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            corr[nt][c] = dec_exp2(m[nt][c] - top[nt][c]);
                            l[nt][c] *= corr[nt][c];
                            m[nt][c] = top[nt][c];
                        }
                    rescale(corr);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const float base = S::P_LOG2 - m[nt][c];
#pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            sh[h][nt][c] = dec_exp2(fmaf(sh[h][nt][c], scale[nt][c], base));
                            sh[h][nt][c + 2] = dec_exp2(fmaf(sh[h][nt][c + 2], scale[nt][c], base));
                            l[nt][c] += sh[h][nt][c] + sh[h][nt][c + 2];
                        }
                    }
                if constexpr (FMT == YUUKA_KV_F16) {
#pragma unroll
                    for (int h = 0; h < HALVES; h++) fragments(h, 1.0f, 1.0f);
                } else if constexpr (S::IS_F8) {
                    const uint32_t bits = dec_lds(ks + S::K16 * HALVES + 4 * KEYS + 4 * (lane & (KEYS - 1))) & 0x7fffffffu;  // a lane to a key, or two
                    v_least = min(v_least, bits - 1);
                    const float inv = take_v_scale(bits);
#pragma unroll
                    for (int h = 0; h < HALVES; h++) fragments(h, vd[h][0] * inv, vd[h][1] * inv);
                }
            }

            // ---- V: sums
            dec_wait<AHEAD - 1>();
            __syncwarp();  // (lanes read what others have copied, and copy over what others have read)
            if constexpr (AHEAD & 1) fetch(std::false_type());
            else fetch(std::true_type());
            const uint32_t vs = take;
            take = take + S::SLOT == ring + S::RING ? ring : take + S::SLOT;

            if (keys > 0) {
                if constexpr (S::IS_F32) {
#pragma unroll
                    for (int half = 0; half < HALVES; half++) {
                        // probabilities in f32 change hands as two 16-bit halves; lane (g, t) then has keys 2t, 2t + 1 (and + 8) of column g
                        uint32_t pk[4], pl[4];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t x = __float_as_uint(sh[half][0][2 * h]), y = __float_as_uint(sh[half][0][2 * h + 1]);
                            const uint32_t low = dec_transpose(__byte_perm(x, y, 0x5410)), high = dec_transpose(__byte_perm(x, y, 0x7632));
                            pk[2 * h] = __byte_perm(low, high, 0x5410);
                            pk[2 * h + 1] = __byte_perm(low, high, 0x7632);
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) pl[i] = dec_rest(pk[i]);
#pragma unroll
                        for (int c = 0; c < CHUNKS; c++) {
                            uint32_t v[4][4];
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint4 r = dec_lds4(vs + half * S::V16 + S::v_piece(2 * t + (k & 1) + 8 * (k >> 1), 8 * c + g));
                                v[k][0] = r.x; v[k][1] = r.y; v[k][2] = r.z; v[k][3] = r.w;
                            }
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                float d[4] = {0.f, 0.f, 0.f, 0.f};  // (summed on its own, as in add_values; small terms first)
#pragma unroll
                                for (int h = 0; h < 2; h++) {
                                    const uint32_t a[4] = {v[2 * h][2 * j], v[2 * h][2 * j + 1], v[2 * h + 1][2 * j], v[2 * h + 1][2 * j + 1]};
                                    uint32_t al[4];
#pragma unroll
                                    for (int i = 0; i < 4; i++) al[i] = dec_rest(a[i]);
                                    dec_mma8(d, al[0], al[1], al[2], al[3], pk[2 * h], pk[2 * h + 1]);
                                    dec_mma8(d, a[0], a[1], a[2], a[3], pl[2 * h], pl[2 * h + 1]);
                                }
#pragma unroll
                                for (int h = 0; h < 2; h++)
                                    dec_mma8(d, v[2 * h][2 * j], v[2 * h][2 * j + 1], v[2 * h + 1][2 * j], v[2 * h + 1][2 * j + 1], pk[2 * h], pk[2 * h + 1]);
#pragma unroll
                                for (int e = 0; e < 4; e++) o[0][c][j][e] += d[e];
                            }
                        }
                    }
                } else if constexpr (S::IS_Q8) {
                    // where the rows of keys 2t + (k & 1) + 8 (k >> 1) begin
                    const uint32_t starts = vs + S::V16 * HALVES;
                    uint32_t row_at[HALVES][4];
#pragma unroll
                    for (int h = 0; h < HALVES; h++)
#pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            const int key = 16 * h + 2 * t + 8 * (k >> 1);
                            const uint2 start = S::Q8_STARTS ? dec_lds2(starts + 4 * key) : make_uint2(0, 0);
                            row_at[h][k] = vs + key * S::Q8_ROW + start.x;
                            row_at[h][k + 1] = vs + (key + 1) * S::Q8_ROW + start.y;
                        }
                    // scales of V: of keys g and g + 8, block by block, into the probabilities
                    float d[HALVES][2][HD / 32];
#pragma unroll
                    for (int h = 0; h < HALVES; h++)
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const int key = 16 * h + g + 8 * k;
                            const uint32_t at = vs + key * S::Q8_ROW + (S::Q8_STARTS ? dec_lds(starts + 4 * key) : 0);
#pragma unroll
                            for (int blk = 0; blk < HD / 32; blk++) d[h][k][blk] = __half2float(__ushort_as_half((unsigned short)dec_lds_u16(at + 34 * blk)));
                        }
                    // the largest and the smallest: a lane to a key, or to half of one's blocks
                    uint32_t largest = 0;
                    {
                        constexpr int EACH = HD / 32 * KEYS / 32;
                        const int key = lane & (KEYS - 1);
                        const uint32_t at = vs + key * S::Q8_ROW + 34 * EACH * (lane / KEYS) + (S::Q8_STARTS ? dec_lds(starts + 4 * key) : 0);
#pragma unroll
                        for (int i = 0; i < EACH; i++) {
                            const uint32_t bits = dec_lds_u16(at + 34 * i) & 0x7fffu;
                            largest = max(largest, bits);
                            v_least = min(v_least, bits - 1);
                        }
                    }
                    const float inv = take_v_scale(__float_as_uint(__half2float(__ushort_as_half((unsigned short)largest))));
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++) {
                        uint32_t a[2][HALVES][4];
#pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            fragments(h, d[h][0][c] * inv, d[h][1][c] * inv);
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint32_t at = row_at[h][k] + 68 * (c >> 1);
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
                                a[j][h][0] = dec_int8<0>(j ? x23 : x01);
                                a[j][h][1] = dec_int8<1>(j ? x23 : x01);
                                a[j][h][2] = dec_int8<0>(j ? y23 : y01);
                                a[j][h][3] = dec_int8<1>(j ? y23 : y01);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) add_values(o[nt][c][j], nt, a[j], pb);
                    }
                } else if constexpr (S::IS_F8) {
                    constexpr int WORDS = S::F8_V / 4;
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++) {
                        uint32_t v[HALVES][4][WORDS];
#pragma unroll
                        for (int h = 0; h < HALVES; h++)
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const int key = 2 * t + (k & 1) + 8 * (k >> 1);
                                const uint32_t at = vs + h * S::V16 + S::v_piece(key, WORDS == 4 ? 8 * c + g : g >> 1) + (WORDS == 4 ? 0 : 8 * (g & 1));
                                if constexpr (WORDS == 4) {
                                    const uint4 r = dec_lds4(at);
                                    v[h][k][0] = r.x; v[h][k][1] = r.y; v[h][k][2] = r.z; v[h][k][3] = r.w;
                                } else {
                                    const uint2 r = dec_lds2(at);
                                    v[h][k][0] = r.x; v[h][k][1] = r.y;
                                }
                            }
#pragma unroll
                        for (int w = 0; w < WORDS; w++)
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                uint32_t a[HALVES][4];
#pragma unroll
                                for (int h = 0; h < HALVES; h++) {
                                    // bytes of two keys next to one another: values of one dimension
                                    const uint2 x = dec_e4m3(__byte_perm(v[h][0][w], v[h][1][w], j ? 0x7362 : 0x5140));
                                    const uint2 y = dec_e4m3(__byte_perm(v[h][2][w], v[h][3][w], j ? 0x7362 : 0x5140));
                                    a[h][0] = x.x; a[h][1] = x.y; a[h][2] = y.x; a[h][3] = y.y;
                                }
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) add_values(o[nt][c][2 * w + j], nt, a, pb);
                            }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < CHUNKS; c++) {
                        uint32_t v[HALVES][4][4];
#pragma unroll
                        for (int h = 0; h < HALVES; h++)
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint4 r = dec_lds4(vs + h * S::V16 + S::v_piece(2 * t + (k & 1) + 8 * (k >> 1), 8 * c + g));
                                v[h][k][0] = r.x; v[h][k][1] = r.y; v[h][k][2] = r.z; v[h][k][3] = r.w;
                            }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint32_t a[HALVES][4];
#pragma unroll
                            for (int h = 0; h < HALVES; h++)
#pragma unroll
                                for (int i = 0; i < 4; i++) a[h][i] = __byte_perm(v[h][i & 2][j], v[h][(i & 2) + 1][j], i & 1 ? 0x7632 : 0x5410);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) add_values(o[nt][c][j], nt, a, pb);
                        }
                    }
                }
            }

            // ---- the end of the unit or of the run
            const bool ends = use.left == 1;
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
                [[maybe_unused]] bool far = false;  // the second kernel does it again
                if constexpr (S::IS_Q8 || S::IS_F8) {  // (for a scale that is not finite as well: it shall make the dimensions that it scales NaN, and no others)
                    const float least = S::IS_F8 ? __uint_as_float(v_least + 1) : __half2float(__ushort_as_half((unsigned short)(v_least + 1)));
                    far = __any_sync(0xffffffffu, (v_least != ~0u && least * (float)(1 << S::FAR_LOG2) < v_scale) || !(v_scale < 1.7e38f));
                }
                const DecodeHeads h = decode_heads(p, unit);
                if (ends && from_start) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int col = nt * 8 + 2 * t + e;
                            if (col >= h.count) continue;
                            const float inv = l[nt][e] == 0.0f ? 0.0f : v_scale / l[nt][e];
                            // a lane's dimensions of a chunk are neighbours (two and two of Q8_0's even blocks)
                            constexpr int RUN = S::IS_Q8 ? 2 : DPL;
                            DecodeRaw<WIDE, RUN> gates[CHUNKS * DPL / RUN];
                            if (p.gate) {
                                const int64_t at = use.b * p.q_row + (h.first + col) * p.q_head;
#pragma unroll
                                for (int i = 0; i < CHUNKS * DPL / RUN; i++)
                                    gates[i].load(p.gate, at + S::out_dim(i * RUN / DPL, i * RUN % DPL / 2, g));
                            }
#pragma unroll
                            for (int i = 0; i < CHUNKS * DPL / RUN; i++) {
                                const int c = i * RUN / DPL, j0 = i * RUN % DPL / 2;
                                float x[RUN];
#pragma unroll
                                for (int j = 0; j < RUN; j++) x[j] = o[nt][c][j0 + j / 2][e + 2 * (j & 1)] * inv;
                                if (p.gate) {
                                    float f[RUN];
                                    dec_gates<WIDE, RUN>(p, gates[i], f);
#pragma unroll
                                    for (int j = 0; j < RUN; j++) x[j] *= f[j];
                                }
                                dec_write<WIDE, RUN>(p, use.b, h.first + col, S::out_dim(c, j0, g), x);
                            }
                            if (g == 0) dec_write_lse(p, use.b, h.first + col, m[nt][e] - S::P_LOG2, l[nt][e]);
                        }
                    again |= far;
                } else {
                    // what other teams share: a row begun earlier (head), or one begun here that goes on (tail)
                    float * const part = p.partial + (((size_t)team * units + unit) * 2 + from_start) * S::PART_FLOATS;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int col = nt * 8 + 2 * t + e;
                            if (col >= h.count) continue;
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                for (int j = 0; j < DPL / 2; j++)
                                    *reinterpret_cast<float2 *>(part + col * HD + S::out_dim(c, j, g)) =
                                        make_float2(o[nt][c][j][e] * v_scale, o[nt][c][j][e + 2] * v_scale);
                            if (g == 0) {
                                part[COLS * HD + col] = m[nt][e] - S::P_LOG2;  // what 1 in l stands for, as the exponentials had it
                                part[COLS * HD + COLS + col] = far ? __uint_as_float(__float_as_uint(l[nt][e]) | 0x80000000u) : l[nt][e];
                            }
                        }
                    if (from_start && lane == 0) {
                        const int last = (int)((begin + it + use.left - 1) / share);
                        const int list = last - (int)team < DEC_SHORT_MOST ? DEC_SHORT : DEC_LONG;
                        const int at = atomicAdd(p.counters + list, 1);
                        if (at < DEC_WARPS) p.joins[list * DEC_WARPS + at] = make_int4(use.b, (int)unit, (int)team, last);
                    }
                }
                fresh = true;
            }
            use.next(p);
        }
        dec_wait<0>();
        if constexpr (S::IS_Q8 || S::IS_F8)
            if (again && lane == 0) {
                const int at = atomicAdd(p.counters + DEC_FAR, 1);
                if (at < DEC_FAR_MOST) p.far[at] = make_int2((int)unit, (int)team);
            }
    }
}

// Q8_0 and F8 once more, in f32 throughout: rows whose scales of V lie far apart, for which f16 probabilities in units of the largest
// scale have too few bits. A key that weighs nothing may have the largest scale, so the unit would have to follow the weighted scales, by
// head and block of dimensions: with such maxima, or with these sums inside the kernel's own loop, ordinary data took 2 to 12 % longer.
//
// A row of K or V: the lane's HD / 32 neighbouring dimensions of a head.
template <int FMT, int HD> __device__ __forceinline__ void decode_row(const uint8_t * row, const PagedCache & c, int kv_head, float (&x)[HD / 32]) {
    constexpr int DIMS = HD / 32;
    const int dim = (threadIdx.x & 31) * DIMS;
    if constexpr (FMT == YUUKA_KV_Q8_0) {
        const uint8_t * block = row + (kv_head * (HD / 32) + dim / 32) * 34;
        const float scale = __half2float(__ushort_as_half(__ldg(reinterpret_cast<const unsigned short *>(block))));
#pragma unroll
        for (int i = 0; i < DIMS; i += 2) {
            const unsigned pair = __ldg(reinterpret_cast<const unsigned short *>(block + 2 + dim % 32 + i));
            x[i] = scale * (float)(int8_t)pair;
            x[i + 1] = scale * (float)(int8_t)(pair >> 8);
        }
    } else {
        const float scale = __ldg(reinterpret_cast<const float *>(row + c.kv_heads * HD) + kv_head);
#pragma unroll
        for (int i = 0; i < DIMS; i += 2) {
            const float2 v = dec_unpack(dec_e4m3(__ldg(reinterpret_cast<const unsigned short *>(row + kv_head * HD + dim + i))).x);
            x[i] = scale * v.x;
            x[i + 1] = scale * v.y;
        }
    }
}
// What a warp makes of a few query heads of a KV head and keys begin .. end - 1 of a sequence: the lane's dimensions of the sums, maximum
// and sum of the probabilities (without the factor that the other kernel's carry). As few heads at once as leave the joins their registers.
template <int HD> constexpr int DEC_AT_ONCE = HD == 256 ? 1 : 2;
template <int HD> struct DecodeColumns {
    float o[DEC_AT_ONCE<HD>][HD / 32], m[DEC_AT_ONCE<HD>], l[DEC_AT_ONCE<HD>];
};
template <int FMT, int HD, bool WIDE>
__device__ __forceinline__ void decode_columns(const DecodeParams & p, int b, int seq, int head, int heads, int kv_head, int begin, int end, DecodeColumns<HD> & result) {
    constexpr int DIMS = HD / 32, A = DEC_AT_ONCE<HD>, FLIGHT = 4;  // keys whose loads are in flight
    const int lane = threadIdx.x & 31, dim = lane * DIMS;
    const PagedCache & c = p.cache;
    const int32_t * const table = c.tables + (int64_t)seq * c.table_stride;
    float q[A][DIMS], o[A][DIMS], m[A], l[A];
#pragma unroll
    for (int a = 0; a < A; a++) {
        DecodeRaw<WIDE, DIMS> raw;
        raw.load(p.q, b * p.q_row + (head + min(a, heads - 1)) * p.q_head + dim);
#pragma unroll
        for (int i = 0; i < DIMS; i += 2) {
            const float2 x = raw.pair(i / 2, p.dtype);
            q[a][i] = x.x;
            q[a][i + 1] = x.y;
            o[a][i] = o[a][i + 1] = 0.0f;
        }
        m[a] = DEC_LOWEST;
        l[a] = 0.0f;
    }
#pragma unroll 1
    for (int pos = begin; pos < end; pos += 32) {
        const int n = min(32, end - pos), mine = lane < n ? kv_slot(c, table, pos + lane) : 0;
        float s[A], sum[A][DIMS];
#pragma unroll
        for (int a = 0; a < A; a++) s[a] = lane < n ? __uint_as_float(0x7fffffffu) : -INFINITY;  // (NaN stays for a bad block)
#pragma unroll 1
        for (int k = 0; k < n; k += FLIGHT) {  // (a lane behind the last key has row 0, and what comes of it goes nowhere)
            float x[FLIGHT][DIMS];
#pragma unroll
            for (int i = 0; i < FLIGHT; i++) decode_row<FMT, HD>(c.k + (int64_t)max(__shfl_sync(0xffffffffu, mine, k + i), 0) * c.row_bytes, c, kv_head, x[i]);
#pragma unroll
            for (int i = 0; i < FLIGHT; i++)
#pragma unroll
                for (int a = 0; a < A; a++) {
                    float dot = 0.0f;
#pragma unroll
                    for (int d = 0; d < DIMS; d++) dot = fmaf(q[a][d], x[i][d], dot);
#pragma unroll
                    for (int w = 16; w > 0; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
                    if (lane == k + i && lane < n && mine >= 0) s[a] = dot * p.scale_log2;
                }
        }
#pragma unroll
        for (int a = 0; a < A; a++) {
            float top = s[a];
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            top = fmaxf(top, m[a]);
            const float corr = exp2f(m[a] - top);
            m[a] = top;
            s[a] = exp2f(s[a] - top);
            float part = s[a];
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) part += __shfl_xor_sync(0xffffffffu, part, w);
            l[a] = fmaf(l[a], corr, part);
#pragma unroll
            for (int d = 0; d < DIMS; d++) {
                o[a][d] *= corr;
                sum[a][d] = 0.0f;
            }
        }
#pragma unroll 1
        for (int k = 0; k < n; k += FLIGHT) {
            float x[FLIGHT][DIMS];
#pragma unroll
            for (int i = 0; i < FLIGHT; i++) decode_row<FMT, HD>(c.v + (int64_t)max(__shfl_sync(0xffffffffu, mine, k + i), 0) * c.row_bytes, c, kv_head, x[i]);
#pragma unroll
            for (int i = 0; i < FLIGHT; i++)
#pragma unroll
                for (int a = 0; a < A; a++) {
                    const float w = __shfl_sync(0xffffffffu, s[a], k + i);
                    if (k + i < n)
#pragma unroll
                        for (int d = 0; d < DIMS; d++) sum[a][d] = fmaf(w, x[i][d], sum[a][d]);
                }
        }
#pragma unroll
        for (int a = 0; a < A; a++)
#pragma unroll
            for (int d = 0; d < DIMS; d++) o[a][d] += sum[a][d];  // (32 keys on their own: fewer roundings of the whole sum)
    }
#pragma unroll
    for (int a = 0; a < A; a++) {
#pragma unroll
        for (int d = 0; d < DIMS; d++) result.o[a][d] = o[a][d];
        result.m[a] = m[a];
        result.l[a] = l[a];
    }
}
// The result of a head whose sums are complete, in the lanes of a warp.
template <int HD, bool WIDE> __device__ __forceinline__ void decode_column_write(const DecodeParams & p, int b, int head, float (&o)[HD / 32], float m, float l) {
    constexpr int DIMS = HD / 32;
    const int lane = threadIdx.x & 31, dim = lane * DIMS;
    float f[DIMS];
    if (p.gate) {
        DecodeRaw<WIDE, DIMS> raw;
        raw.load(p.gate, b * p.q_row + head * p.q_head + dim);
        dec_gates<WIDE, DIMS>(p, raw, f);
    }
#pragma unroll
    for (int i = 0; i < DIMS; i++) o[i] = l == 0.0f ? 0.0f : o[i] / l * (p.gate ? f[i] : 1.0f);
    dec_write<WIDE, DIMS>(p, b, head, dim, o);
    if (lane == 0) dec_write_lse(p, b, head, m, l);
}
// DEC_AT_ONCE heads of a row that several teams share, by all warps of a CTA: each takes some of the keys. `store`: shared memory.
template <int HD> constexpr int DEC_STORE = 8 * DEC_AT_ONCE<HD> * (HD + 2);  // floats
template <int FMT, int HD, bool WIDE> __device__ __forceinline__ void decode_row_again(const DecodeParams & p, int b, int unit, int col, float * store) {
    constexpr int DIMS = HD / 32, A = DEC_AT_ONCE<HD>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;  // (eight)
    const DecodeHeads heads = decode_heads(p, unit);
    const DecodeSpan span = decode_span(p, b, 16);
    const int each = ((span.end - span.first + 32 * warps - 1) / (32 * warps)) * 32, begin = min(span.first + warp * each, span.end);
    DecodeColumns<HD> r;
    decode_columns<FMT, HD, WIDE>(p, b, max(span.seq, 0), heads.first + col, min(A, heads.count - col), heads.kv_head, begin, min(begin + each, span.end), r);
    __syncthreads();  // (the store's last use)
#pragma unroll
    for (int a = 0; a < A; a++) {
        float * const mine = store + (warp * A + a) * (HD + 2);
#pragma unroll
        for (int i = 0; i < DIMS; i++) mine[lane * DIMS + i] = r.o[a][i];
        if (lane == 0) {
            mine[HD] = r.m[a];
            mine[HD + 1] = r.l[a];
        }
    }
    __syncthreads();
    if (warp < A && col + warp < heads.count) {
        float o[DIMS], m = DEC_LOWEST, l = 0.0f;
        for (int w = 0; w < warps; w++) m = fmaxf(m, store[(w * A + warp) * (HD + 2) + HD]);
#pragma unroll
        for (int i = 0; i < DIMS; i++) o[i] = 0.0f;
        for (int w = 0; w < warps; w++) {
            const float * const part = store + (w * A + warp) * (HD + 2);
            const float f = exp2f(part[HD] - m);
            l = fmaf(f, part[HD + 1], l);
#pragma unroll
            for (int i = 0; i < DIMS; i++) o[i] = fmaf(f, part[lane * DIMS + i], o[i]);
        }
        decode_column_write<HD, WIDE>(p, b, heads.first + col + warp, o, m, l);
    }
    __syncthreads();
}
// Whole rows of a run: the warps of the CTA take them in turn.
template <int FMT, int HD, int NT, bool WIDE> __device__ __forceinline__ void decode_again(const DecodeParams & p, unsigned unit, unsigned team) {
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    constexpr int KEYS = S::KEYS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const PagedCache & c = p.cache;
    const unsigned units = c.kv_heads * p.head_tiles, teams = max(p.warps / units, 1u);
    if (unit >= units || team >= teams) return;
    unsigned total = 0;
    for (int b = lane; b < p.batch; b += 32) total += decode_span(p, b, KEYS).tiles;
    total = __reduce_add_sync(0xffffffffu, total);
    const unsigned share = (total + teams - 1) / teams, begin = team * share;
    if (begin >= total) return;
    const DecodeHeads heads = decode_heads(p, unit);
    DecodeCursor<KEYS> use;
    use.seek(p, begin);
    unsigned left = min(share, total - begin);
    for (int turn = 0; left > 0 && use.b < p.batch; turn++) {
        const unsigned tiles = min((unsigned)use.left, left);
        if (use.left == use.tiles && tiles == (unsigned)use.tiles && use.end > use.first && turn % warps == warp) {
            // The row's largest and smallest scale of V but zero, as the other kernel has seen them. (Half its ratio: its unit is the next
            // power of two.)
            const int32_t * const table = c.tables + (int64_t)use.seq * c.table_stride;
            float largest = 0.0f, least = INFINITY;
            bool wild = false;
            for (int pos = use.first + lane; pos < use.end; pos += 32) {
                const int slot = kv_slot(c, table, pos);
                if (slot < 0) continue;
                const uint8_t * const row = c.v + (int64_t)slot * c.row_bytes;
                for (int i = 0; i < (FMT == YUUKA_KV_Q8_0 ? HD / 32 : 1); i++) {
                    float d;
                    if constexpr (FMT == YUUKA_KV_Q8_0)
                        d = fabsf(__half2float(__ushort_as_half(__ldg(reinterpret_cast<const unsigned short *>(row + (heads.kv_head * (HD / 32) + i) * 34)))));
                    else d = fabsf(__ldg(reinterpret_cast<const float *>(row + c.kv_heads * HD) + heads.kv_head));
                    wild |= !(d < 1.7e38f);
                    largest = fmaxf(largest, d);
                    if (d != 0.0f) least = fminf(least, d);
                }
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) {
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, w));
                least = fminf(least, __shfl_xor_sync(0xffffffffu, least, w));
            }
            if (__any_sync(0xffffffffu, wild || least * (float)(1 << (S::FAR_LOG2 - 1)) < largest || least < 1.2e-38f))
                for (int col = 0; col < heads.count; col += DEC_AT_ONCE<HD>) {
                    const int n = min(DEC_AT_ONCE<HD>, heads.count - col);
                    DecodeColumns<HD> r;
                    decode_columns<FMT, HD, WIDE>(p, use.b, use.seq, heads.first + col, n, heads.kv_head, use.first, use.end, r);
#pragma unroll
                    for (int a = 0; a < DEC_AT_ONCE<HD>; a++)
                        if (a < n) decode_column_write<HD, WIDE>(p, use.b, heads.first + col + a, r.o[a], r.m[a], r.l[a]);
                }
        }
        left -= tiles;
        if (++use.b < p.batch) use.row(p);
        use.pos = use.first;
        use.left = use.tiles;
    }
}

// The units that several teams share. Few partials: a CTA takes a unit, a warp a column, a lane HD / 32 dimensions. Many: a CTA
// takes 32 dimensions of a column at a time; groups of 8 threads take every 32nd partial, so that many loads are in flight, and
// are added in their order.
constexpr int JOIN_THREADS = 256, JOIN_CTAS_SM = 4, JOIN_LANES = 8, JOIN_GROUPS = JOIN_THREADS / JOIN_LANES;
template <int FMT, int HD, int NT, bool WIDE>  // (FMT: Q8_0, F8 or any other)
__global__ void __launch_bounds__(JOIN_THREADS, 2) attention_decode_join_kernel(const __grid_constant__ DecodeParams p) {
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    constexpr int COLS = S::COLS, PART = COLS * (HD + 2), SLICES = HD / (4 * JOIN_LANES), DIMS = HD / 32;
    constexpr bool FAR = S::IS_Q8 || S::IS_F8;  // (joins of which a part's sums have a sign are rows to be done again)
    [[maybe_unused]] bool again = false;        // this warp has met one
    __shared__ float factor[FAR && DEC_STORE<HD> > DEC_WARPS ? DEC_STORE<HD> : DEC_WARPS], reduce[2][JOIN_THREADS / 32];
    __shared__ float4 sums[JOIN_GROUPS][JOIN_LANES];
    pdl_entry();
    const int tid = threadIdx.x, units = p.cache.kv_heads * p.head_tiles, group = tid / JOIN_LANES;
    const int few = min(p.counters[DEC_SHORT], DEC_WARPS), jobs = min(p.counters[DEC_LONG], DEC_WARPS) * COLS * SLICES,
              runs = FAR ? min(p.counters[DEC_FAR], DEC_FAR_MOST) : 0;
#pragma unroll 1
    for (int job = blockIdx.x; job < few; job += gridDim.x) {
        const int4 join = p.joins[job];
        if (!decode_join_sound(p, join)) continue;
        const DecodeHeads h = decode_heads(p, join.y);
        const int n = join.w - join.z + 1, lane = tid & 31, dim = lane * DIMS;
        const float * first = p.partial + ((size_t)join.z * units + join.y) * 2 * PART;
        const int64_t stride = (int64_t)units * 2 * PART;
        for (int col = tid >> 5; col < h.count; col += JOIN_THREADS / 32) {
            const float * mine = first + lane * stride + (lane ? 0 : PART) + COLS * HD + col;
            const float ms = lane < n ? mine[0] : -INFINITY, ls = lane < n ? mine[COLS] : 0.0f;
            if constexpr (FAR)
                if (__any_sync(0xffffffffu, (int)__float_as_uint(ls) < 0)) {
                    again = true;
                    break;
                }
            DecodeRaw<WIDE, DIMS> raw;
            if (p.gate) raw.load(p.gate, join.x * p.q_row + (h.first + col) * p.q_head + dim);
            float m = ms, x[DIMS];
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
            const float f = lane < n ? exp2f(ms - m) : 0.0f;
            float l = f * ls;
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
            for (int i = 0; i < DIMS; i++) x[i] = 0.0f;
            constexpr int FLIGHT = 32 / DIMS;  // partials whose loads are in flight
#pragma unroll 1
            for (int k0 = 0; k0 < n; k0 += FLIGHT) {
                DecodeRaw<true, DIMS> o[FLIGHT];
#pragma unroll
                for (int i = 0; i < FLIGHT; i++) {
                    const int k = min(k0 + i, n - 1);
                    o[i].fetch(first + k * stride + (k ? 0 : PART) + col * HD + dim);
                }
#pragma unroll
                for (int i = 0; i < FLIGHT; i++) {
                    const float fk = k0 + i < n ? __shfl_sync(0xffffffffu, f, k0 + i) : 0.0f;
                    if (k0 + i < n)
#pragma unroll
                        for (int d = 0; d < DIMS; d++) x[d] = fmaf(fk, __uint_as_float(o[i].w[d]), x[d]);
                }
            }
            float gates[DIMS];
            if (p.gate) dec_gates<WIDE, DIMS>(p, raw, gates);
#pragma unroll
            for (int d = 0; d < DIMS; d++) x[d] = l == 0.0f ? 0.0f : x[d] / l * (p.gate ? gates[d] : 1.0f);
            dec_write<WIDE, DIMS>(p, join.x, h.first + col, dim, x);
            if (lane == 0) dec_write_lse(p, join.x, h.first + col, m, l);
        }
    }
#pragma unroll 1
    for (int job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int4 join = p.joins[DEC_WARPS + job / (COLS * SLICES)];
        if (!decode_join_sound(p, join)) continue;
        const int col = job / SLICES % COLS, dim = 4 * (job % SLICES * JOIN_LANES + tid % JOIN_LANES);
        const DecodeHeads h = decode_heads(p, join.y);
        if (col >= h.count) continue;
        const int n = join.w - join.z + 1;  // partials: the tail of the first team and the heads of the following ones
        const float * first = p.partial + ((size_t)join.z * units + join.y) * 2 * PART;
        const int64_t stride = (int64_t)units * 2 * PART;
        auto part = [&](int k) { return first + k * stride + (k ? 0 : PART); };
        float gate[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if (p.gate && group == 0) {
            DecodeRaw<WIDE, 4> raw;
            raw.load(p.gate, join.x * p.q_row + (h.first + col) * p.q_head + dim);
            dec_gates<WIDE, 4>(p, raw, gate);
        }
        // the first loads of sums are on their way while the statistics are made
        float4 o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = group + i * JOIN_GROUPS;
            o[i] = k < n ? *reinterpret_cast<const float4 *>(part(k) + col * HD + dim) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float m = -INFINITY;
        for (int k = tid; k < n; k += JOIN_THREADS) m = fmaxf(m, part(k)[COLS * HD + col]);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
        if ((tid & 31) == 0) reduce[0][tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; w++) m = fmaxf(m, reduce[0][w]);
        float l = 0.0f;
        [[maybe_unused]] bool far = false;
        for (int k = tid; k < n; k += JOIN_THREADS) {
            const float f = exp2f(part(k)[COLS * HD + col] - m);
            factor[k] = f;
            const float lk = part(k)[COLS * HD + COLS + col];
            if constexpr (FAR) far |= (int)__float_as_uint(lk) < 0;
            l = fmaf(f, lk, l);
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
        if ((tid & 31) == 0) reduce[1][tid >> 5] = l;
        if constexpr (FAR) {
            if (__syncthreads_or(far)) {
                again = true;
                continue;
            }
        } else {
            __syncthreads();
        }
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; w++) l += reduce[1][w];
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int k0 = group; k0 < n; k0 += 4 * JOIN_GROUPS) {
            if (k0 != group) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int k = k0 + i * JOIN_GROUPS;
                    o[i] = k < n ? *reinterpret_cast<const float4 *>(part(k) + col * HD + dim) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = k0 + i * JOIN_GROUPS;
                if (k >= n) continue;
                const float f = factor[k];
                x.x = fmaf(f, o[i].x, x.x);
                x.y = fmaf(f, o[i].y, x.y);
                x.z = fmaf(f, o[i].z, x.z);
                x.w = fmaf(f, o[i].w, x.w);
            }
        }
        sums[group][tid % JOIN_LANES] = x;
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int i = 1; i < JOIN_GROUPS; i++) {
                const float4 y = sums[i][tid];
                x.x += y.x;
                x.y += y.y;
                x.z += y.z;
                x.w += y.w;
            }
            if (l == 0.0f) x = make_float4(0.f, 0.f, 0.f, 0.f), l = 1.0f, m = -INFINITY;  // (all scores are -infinity)
            dec_write<WIDE, 4>(p, join.x, h.first + col, dim, {x.x / l * gate[0], x.y / l * gate[1], x.z / l * gate[2], x.w / l * gate[3]});
            if (dim == 0) dec_write_lse(p, join.x, h.first + col, m, l);
        }
        __syncthreads();
    }
    // Rows to be done again, behind the loops: inside them they took registers of theirs
    if constexpr (FAR) {
#pragma unroll 1
        for (int job = blockIdx.x; job < runs; job += gridDim.x) decode_again<FMT, HD, NT, WIDE>(p, p.far[job].x, p.far[job].y);
        if (__syncthreads_or(again)) {  // (the jobs that this CTA has had)
            auto is_far = [&](const int4 & join) {
                bool far = false;
                for (int k = tid; k <= join.w - join.z; k += JOIN_THREADS)
                    far |= (int)__float_as_uint(p.partial[(((size_t)(join.z + k) * units + join.y) * 2 + (k ? 0 : 1)) * PART + COLS * HD + COLS]) < 0;
                return __syncthreads_or(far) != 0;
            };
#pragma unroll 1
            for (int job = blockIdx.x; job < few; job += gridDim.x) {
                const int4 join = p.joins[job];
                if (!decode_join_sound(p, join) || !is_far(join)) continue;
                const int count = decode_heads(p, join.y).count;
                for (int col = 0; col < count; col += DEC_AT_ONCE<HD>) decode_row_again<FMT, HD, WIDE>(p, join.x, join.y, col, factor);
            }
            // the job of a long join's first dimensions, and of the first of so many columns, does them all
#pragma unroll 1
            for (int job = blockIdx.x; job < jobs; job += gridDim.x) {
                const int4 join = p.joins[DEC_WARPS + job / (COLS * SLICES)];
                const int col = job / SLICES % COLS;
                if (!decode_join_sound(p, join) || job % SLICES != 0 || col % DEC_AT_ONCE<HD> != 0 || col >= decode_heads(p, join.y).count || !is_far(join)) continue;
                decode_row_again<FMT, HD, WIDE>(p, join.x, join.y, col, factor);
            }
        }
    }
    // the last CTA leaves the counters as the call found them
    __syncthreads();
    if (tid == 0 && atomicAdd(p.counters + DEC_DONE, 1) == (int)gridDim.x - 1) p.counters[DEC_SHORT] = p.counters[DEC_LONG] = p.counters[DEC_FAR] = p.counters[DEC_DONE] = 0;
}

// Launches for one format on a device with `sms` multiprocessors.
void launch_decode_f32(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int sms);
void launch_decode_f16(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int sms);
void launch_decode_q8_0(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int sms);
void launch_decode_f8(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int sms);

template <int FMT, int HD, int NT, bool WIDE> void launch_decode_as(cudaStream_t s, DecodeParams p, int sms) {
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    const int ctas = sms * S::RESIDENT;
    YK_REQUIRE(ctas * S::W <= DEC_WARPS && ctas * S::W * 2 * S::PART_FLOATS * sizeof(float) <= DEC_PARTIAL_BYTES, YUUKA_ERR_UNSUPPORTED,
               "attention_decode: %d multiprocessors", sms);
    auto kern = attention_decode_kernel<FMT, HD, NT, WIDE>;
    YK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::LAYOUT_BYTES));
    p.warps = ctas * S::W;
    launch_k(kern, (unsigned)ctas, S::W * 32, S::LAYOUT_BYTES, s, p);
    constexpr int JOIN = S::IS_Q8 || S::IS_F8 ? FMT : YUUKA_KV_F16;
    launch_k(attention_decode_join_kernel<JOIN, HD, NT, WIDE>, (unsigned)(sms * JOIN_CTAS_SM), JOIN_THREADS, 0, s, p);
}
template <int FMT, int HD, int NT> void launch_decode_tiles(cudaStream_t s, const DecodeParams & p, int sms) {
    if (p.dtype == YUUKA_DTYPE_F32) launch_decode_as<FMT, HD, NT, true>(s, p, sms);
    else launch_decode_as<FMT, HD, NT, false>(s, p, sms);
}
template <int FMT, int NT> void launch_decode_dims(cudaStream_t s, const DecodeParams & p, int head_dim, int sms) {
    if (head_dim == 64) launch_decode_tiles<FMT, 64, NT>(s, p, sms);
    else if (head_dim == 128) launch_decode_tiles<FMT, 128, NT>(s, p, sms);
    else launch_decode_tiles<FMT, 256, NT>(s, p, sms);
}

}  // namespace yk
