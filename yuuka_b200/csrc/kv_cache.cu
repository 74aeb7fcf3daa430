// Rows of a paged key-value cache: written in the cache's format, read back as plain numbers (yuuka_kv_write, yuuka_kv_read).
//
// Both move a row once and compute little, so what bounds them is memory: rows * 2 * (numbers + pool row) bytes. A warp takes
// up to 1024 values of a K or V row, 256 at a time (eight per lane, one 16- or 32-byte load), all of its loads in flight before
// the first is used and the row's place looked up once: 30,000 rows of 8 x 128 bf16 take 37 us into F8 (5.0 TB/s), with 256 values
// a warp and a loop over a grid of resident CTAs they took 83. Reading them back takes 38. 256 values hold whole Q8_0 blocks (four
// lanes each) and whole heads (8, 16 or 32 lanes each), so the maxima that the scales come from need shuffles alone.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "kv_cache.cuh"
#include "quant.cuh"

namespace yk {

// ---------------------------------------------------------------------------
// checks of arguments

uint64_t kv_row_bytes(int32_t format, int32_t kv_heads, int32_t head_dim) {
    if (kv_heads < 1 || kv_heads > 1024 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
    const uint64_t n = (uint64_t)kv_heads * head_dim;
    switch (format) {
    case YUUKA_KV_F32: return 4 * n;
    case YUUKA_KV_F16: return 2 * n;
    case YUUKA_KV_Q8_0: return n / 32 * 34;
    case YUUKA_KV_F8: return (n + 4 * (uint64_t)kv_heads + 15) / 16 * 16;
    default: return 0;
    }
}

void check_geometry(const char * op, const yuuka_kv_cache * c) {
    YK_REQUIRE(c->format >= YUUKA_KV_F32 && c->format <= YUUKA_KV_F8, YUUKA_ERR_INVALID_ARGUMENT, "%s: unknown KV format %d", op, c->format);
    YK_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 1024, YUUKA_ERR_INVALID_ARGUMENT, "%s: %d KV heads are not 1..1024", op, c->kv_heads);
    YK_REQUIRE(kv_row_bytes(c->format, c->kv_heads, c->head_dim) > 0, YUUKA_ERR_UNSUPPORTED, "%s: head_dim %d is not 64, 128 or 256", op,
               c->head_dim);
    YK_REQUIRE(c->block_size >= 1 && c->pool_blocks >= 1 && (uint64_t)c->block_size * (uint64_t)c->pool_blocks <= INT_MAX,
               YUUKA_ERR_INVALID_ARGUMENT, "%s: %d blocks of %d rows are not 1..2^31 - 1 rows", op, c->pool_blocks, c->block_size);
    YK_REQUIRE(c->sequences >= 1 && c->table_stride >= 1, YUUKA_ERR_INVALID_ARGUMENT, "%s: %d block tables of %d ids", op, c->sequences,
               c->table_stride);
}

uint64_t span_bytes(uint64_t rows, uint64_t row_stride, uint64_t heads, uint64_t head_stride, uint64_t dim, uint64_t size) {
    const unsigned __int128 n =
        ((unsigned __int128)(rows - 1) * row_stride + (unsigned __int128)(heads - 1) * head_stride + dim) * size;
    return n >> 62 ? UINT64_MAX : (uint64_t)n;
}

void check_range(const char * op, const char * what, const yuuka_buffer * buf, uint64_t offset, uint64_t bytes, uint64_t align,
                 const yuuka_device * dev) {
    YK_REQUIRE(buf, YUUKA_ERR_INVALID_ARGUMENT, "%s: %s is null", op, what);
    YK_REQUIRE(buf->dev->index == dev->index, YUUKA_ERR_INVALID_ARGUMENT, "%s: %s is on device %d, the stream on device %d", op, what,
               buf->dev->index, dev->index);
    YK_REQUIRE(offset <= buf->bytes && bytes <= buf->bytes - offset, YUUKA_ERR_INVALID_ARGUMENT, "%s: %s range exceeds the buffer", op, what);
    check_start(op, what, buf, offset, align);
}

void check_apart(const char * op, const char * a_name, const yuuka_buffer * a, uint64_t a_offset, uint64_t a_bytes, const char * b_name,
                 const yuuka_buffer * b, uint64_t b_offset, uint64_t b_bytes) {
    if (!a || !b) return;
    const uint64_t a0 = (uint64_t)(uintptr_t)a->ptr + a_offset, b0 = (uint64_t)(uintptr_t)b->ptr + b_offset;
    YK_REQUIRE(a0 + a_bytes <= b0 || b0 + b_bytes <= a0, YUUKA_ERR_INVALID_ARGUMENT, "%s: %s lies over %s", op, a_name, b_name);
}

PagedCache check_cache(const char * op, const yuuka_kv_cache * c, const yuuka_device * dev) {
    check_geometry(op, c);
    const uint64_t rb = kv_row_bytes(c->format, c->kv_heads, c->head_dim), pool = rb * (uint64_t)c->block_size * (uint64_t)c->pool_blocks;
    check_range(op, "the K pool", c->k, c->k_offset, pool, 16, dev);
    check_range(op, "the V pool", c->v, c->v_offset, pool, 16, dev);
    check_range(op, "the block table", c->tables, c->tables_offset, 4ull * (uint64_t)c->sequences * (uint64_t)c->table_stride, 4, dev);
    check_apart(op, "the K pool", c->k, c->k_offset, pool, "the V pool", c->v, c->v_offset, pool);
    PagedCache p;
    p.k = (uint8_t *)c->k->ptr + c->k_offset;
    p.v = (uint8_t *)c->v->ptr + c->v_offset;
    p.tables = (const int32_t *)((const uint8_t *)c->tables->ptr + c->tables_offset);
    p.row_bytes = (int64_t)rb;
    p.format = c->format;
    p.kv_heads = c->kv_heads;
    p.block_size = c->block_size;
    p.pool_blocks = c->pool_blocks;
    p.sequences = c->sequences;
    p.table_stride = c->table_stride;
    p.shift = -1;
    for (int s = 0; s < 31; s++)
        if (c->block_size == 1 << s) p.shift = s;
    p.capacity = (int)std::min<uint64_t>((uint64_t)c->table_stride * (uint64_t)c->block_size, INT_MAX);
    return p;
}

// ---------------------------------------------------------------------------
// kernels

struct MoveParams {
    PagedCache cache;
    uint8_t * k;  // rows of numbers
    uint8_t * v;
    int64_t k_stride, v_stride;  // elements
    const int32_t * pos;
    const int32_t * seq;
    int32_t * status;
    int rows, kv_dim, groups;  // groups of 1024 values in a row
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// Eight neighbouring values as they come from memory.
template <typename T> struct Eight {
    uint4 raw[sizeof(T) / 2];
    __device__ __forceinline__ void load(const void * src) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const T * e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)e[i];
    }
    // largest magnitude; a NaN does not count, or makes it one
    template <bool NANS> __device__ __forceinline__ float largest() const {
        if constexpr (sizeof(T) == 4) {
            const float * e = reinterpret_cast<const float *>(raw);
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) m = NANS ? max_nan(m, fabsf(e[i])) : fmaxf(m, fabsf(e[i]));
            return m;
        } else {
            using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            const Pair * e = reinterpret_cast<const Pair *>(raw);
            if constexpr (NANS) {
                const Pair m = __hmax2_nan(__hmax2_nan(__habs2(e[0]), __habs2(e[1])), __hmax2_nan(__habs2(e[2]), __habs2(e[3])));
                return max_nan((float)m.x, (float)m.y);
            }
            const Pair m = __hmax2(__hmax2(__habs2(e[0]), __habs2(e[1])), __hmax2(__habs2(e[2]), __habs2(e[3])));
            return fmaxf(fmaxf((float)m.x, (float)m.y), 0.0f);
        }
    }
};
template <typename T> __device__ __forceinline__ void store8(T * dst, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 raw;
        T * e = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = (T)x[i];
        *reinterpret_cast<uint4 *>(dst) = raw;
    }
}

// f32 -> f16 bits, half up on the dropped bits. Magnitudes whose result is a normal f16 take one add and a conversion that
// cuts off; the others the codec's own steps.
__device__ __forceinline__ uint16_t half_up(float f) {
    const uint32_t b = __float_as_uint(f), a = b & 0x7fffffffu;
    if (a >= 0x38800000u && a < 0x477ff000u) return __half_as_ushort(__float2half_rz(__uint_as_float(b + 0x1000u)));
    return f32_to_f16_ref(f);
}
// The nearest integers to v / scale, halves away from zero, of the f32 quotients, as bytes. The product with 1 / scale is within
// 2^-22 of the quotient (relative; at most 127.5 in magnitude, so 2^-15 in all): where it is not within 1e-4 of a half it rounds
// to the same integer, which adding 1.5 * 2^23 leaves in the low byte. Others, and NaN, take the quotient itself.
__device__ __forceinline__ uint2 quantize_q8(const float (&v)[8], float scale, float inv) {
    constexpr float MAGIC = 12582912.0f;
    uint32_t q[8];
    bool sure = inv <= 3.0e38f;  // (a scale whose inverse is no finite number)
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float r = fmaf(v[i], inv, MAGIC);
        q[i] = __float_as_uint(r);
        sure &= fabsf(fmaf(v[i], inv, MAGIC - r)) <= 0.4999f;
    }
    if (!sure) {
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = scale != 0.0f ? (uint32_t)(int)round((double)(v[i] / scale)) : 0u;
    }
    return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
}

// Where row r's token lies: the pool row, -1 for a row without a token, -2 for one out of range.
__device__ __forceinline__ int move_slot(const MoveParams & p, int r) {
    const int pos = __ldg(p.pos + r), seq = p.seq ? __ldg(p.seq + r) : r;
    int bad;
    const int slot = kv_token_slot(p.cache, seq, pos, bad);
    if (bad && p.status && (threadIdx.x & 31) == 0) atomicOr(p.status, bad);
    return slot;
}

constexpr int MOVE_WARPS = 8, MOVE_CHUNKS = 4;
constexpr int Q8_CHUNK = 272;  // bytes of 256 values in Q8_0

// A warp's part: row, K or V, values first .. (of up to MOVE_CHUNKS chunks of 256).
struct MoveUnit {
    int r, first, chunks;
    bool is_v;
    __device__ __forceinline__ MoveUnit(const MoveParams & p) {
        const unsigned unit = blockIdx.x * MOVE_WARPS + (threadIdx.x >> 5), parts = 2 * p.groups;
        r = (int)(unit / parts);
        const int rest = (int)(unit - (unsigned)r * parts);
        is_v = rest >= p.groups;
        first = (is_v ? rest - p.groups : rest) * 256 * MOVE_CHUNKS;
        chunks = r < p.rows ? min(MOVE_CHUNKS, (p.kv_dim - first + 255) / 256) : 0;
    }
};

// Words of a chunk of Q8_0 between shared memory and a pool row: rows that are a multiple of 16 bytes long by 16 bytes.
template <bool STORE> __device__ __forceinline__ void move_q8_chunk(uint8_t * stage, uint8_t * row, int values, bool wide) {
    const int lane = threadIdx.x & 31;
    if (wide && values >= 256) {
        if (lane < Q8_CHUNK / 16) {
            if constexpr (STORE) reinterpret_cast<uint4 *>(row)[lane] = reinterpret_cast<const uint4 *>(stage)[lane];
            else reinterpret_cast<uint4 *>(stage)[lane] = __ldg(reinterpret_cast<const uint4 *>(row) + lane);
        }
        return;
    }
    const int words = min(values, 256) / 32 * 34 / 4;
    for (int w = lane; w < words; w += 32) {
        if constexpr (STORE) reinterpret_cast<uint32_t *>(row)[w] = reinterpret_cast<const uint32_t *>(stage)[w];
        else reinterpret_cast<uint32_t *>(stage)[w] = __ldg(reinterpret_cast<const uint32_t *>(row) + w);
    }
}

// The pool is aligned to 16 bytes, a row of Q8_0 to 4: its blocks of 34 bytes are put together in shared memory.
template <int FMT, int HD, typename T>
__global__ void __launch_bounds__(MOVE_WARPS * 32) kv_write_kernel(const MoveParams p) {
    __shared__ __align__(16) uint8_t stage_all[FMT == YUUKA_KV_Q8_0 ? MOVE_WARPS * MOVE_CHUNKS * Q8_CHUNK : 16];
    pdl_entry();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const MoveUnit u(p);
    if (u.chunks == 0) return;
    Eight<T> x[MOVE_CHUNKS];
    const T * src = reinterpret_cast<const T *>(u.is_v ? p.v : p.k) + (int64_t)u.r * (u.is_v ? p.v_stride : p.k_stride) + u.first + lane * 8;
#pragma unroll
    for (int c = 0; c < MOVE_CHUNKS; c++) {
        x[c].zero();
        if (u.first + c * 256 + lane * 8 < p.kv_dim) x[c].load(src + c * 256);
    }
    const int slot = move_slot(p, u.r);
    if (slot < 0) return;  // (the whole warp: one row)
    uint8_t * row = (u.is_v ? p.cache.v : p.cache.k) + (int64_t)slot * p.cache.row_bytes;

    // Scales: every division is made once, by one lane, for all chunks at a time, and handed to the lanes that need it.
    // (amax / 127 and amax / 448 by their inverses: within an ulp of the quotient. Q8_0's scales, f16 in the end, are the quotient's all the
    // same: 127 f32(1 / 127) is 1 - 2^-28, and no f32 lies near enough below 127 times a border of f16's rounding. Whole numbers differ
    // by one from those of a session where a value's quotient is a half, or within an f32 step of one.)
    float scale[MOVE_CHUNKS], inv[MOVE_CHUNKS];
    uint32_t half_scale = 0;  // Q8_0: of block lane (eight of a chunk)
    if constexpr (FMT == YUUKA_KV_Q8_0 || FMT == YUUKA_KV_F8) {
        constexpr int LANES = FMT == YUUKA_KV_Q8_0 ? 4 : HD / 8;  // that share a scale
        static_assert(MOVE_CHUNKS == 4, "the divisions' lanes");
        float amax[MOVE_CHUNKS];
#pragma unroll
        for (int c = 0; c < MOVE_CHUNKS; c++) {
            amax[c] = x[c].template largest<FMT == YUUKA_KV_F8>();
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, amax[c], o);
                amax[c] = FMT == YUUKA_KV_F8 ? max_nan(amax[c], other) : fmaxf(amax[c], other);
            }
        }
        if constexpr (FMT == YUUKA_KV_Q8_0) {
            float mine = 0.0f;
#pragma unroll
            for (int c = 0; c < MOVE_CHUNKS; c++) {
                const float a = __shfl_sync(0xffffffffu, amax[c], 4 * (lane & 7));
                if (lane >> 3 == c) mine = a;
            }
            const float s = mine * (1.0f / 127.0f), r = 1.0f / s;
            half_scale = half_up(s);
#pragma unroll
            for (int c = 0; c < MOVE_CHUNKS; c++) {
                scale[c] = __shfl_sync(0xffffffffu, s, 8 * c + (lane >> 2));
                inv[c] = __shfl_sync(0xffffffffu, r, 8 * c + (lane >> 2));
            }
        } else {
            const int at = lane & (LANES - 1);
            const float mine = (at & 2) ? ((at & 1) ? amax[3] : amax[2]) : ((at & 1) ? amax[1] : amax[0]);
            const float r = (at & 4) ? mine * (1.0f / 448.0f) : 1.0f / mine * 448.0f;
#pragma unroll
            for (int c = 0; c < MOVE_CHUNKS; c++) {
                inv[c] = __shfl_sync(0xffffffffu, r, lane - at + c);
                scale[c] = __shfl_sync(0xffffffffu, r, lane - at + 4 + c);
                if (inv[c] > 3.0e38f) scale[c] = 0.0f;  // (nothing but zeros, or too small for a finite factor)
                if (!(inv[c] <= 3.0e38f)) inv[c] = 0.0f;  // (a NaN among the values makes the scale one)
            }
        }
    }
#pragma unroll
    for (int c = 0; c < MOVE_CHUNKS; c++) {
        if (c >= u.chunks) break;
        const int first = u.first + c * 256 + lane * 8;
        const bool live = first < p.kv_dim;
        float f[8];
        x[c].get(f);
        if constexpr (FMT == YUUKA_KV_F32) {
            if (live) store8(reinterpret_cast<float *>(row) + first, f);
        } else if constexpr (FMT == YUUKA_KV_F16) {
            if (live) {
                uint4 raw;
                uint16_t * e = reinterpret_cast<uint16_t *>(&raw);
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] = half_up(f[i]);
                *reinterpret_cast<uint4 *>(row + 2 * first) = raw;
            }
        } else if constexpr (FMT == YUUKA_KV_Q8_0) {
            const uint2 q = quantize_q8(f, scale[c], inv[c]);
            uint16_t * chunk = reinterpret_cast<uint16_t *>(stage_all + (warp * MOVE_CHUNKS + c) * Q8_CHUNK);
            uint16_t * blk = chunk + (lane >> 2) * 17 + 1 + (lane & 3) * 4;
            blk[0] = (uint16_t)q.x;
            blk[1] = (uint16_t)(q.x >> 16);
            blk[2] = (uint16_t)q.y;
            blk[3] = (uint16_t)(q.y >> 16);
            if (lane >> 3 == c) chunk[(lane & 7) * 17] = (uint16_t)half_scale;
        } else {
            uint2 raw;
            __nv_fp8x2_storage_t * e = reinterpret_cast<__nv_fp8x2_storage_t *>(&raw);
#pragma unroll
            for (int i = 0; i < 4; i++) e[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv[c], f[2 * i + 1] * inv[c]), __NV_SATFINITE, __NV_E4M3);
            if (live) {
                *reinterpret_cast<uint2 *>(row + first) = raw;
                if (first % HD == 0) *reinterpret_cast<float *>(row + p.kv_dim + first / HD * 4) = scale[c];
                // (the zeros behind the scales)
                if (first + 8 == p.kv_dim)
                    for (int at = p.kv_dim + 4 * (p.kv_dim / HD); at < p.cache.row_bytes; at += 4) *reinterpret_cast<uint32_t *>(row + at) = 0;
            }
        }
    }
    if constexpr (FMT == YUUKA_KV_Q8_0) {
        __syncwarp();
        for (int c = 0; c < u.chunks; c++)
            move_q8_chunk<true>(stage_all + (warp * MOVE_CHUNKS + c) * Q8_CHUNK, row + (u.first / 256 + c) * Q8_CHUNK, p.kv_dim - u.first - c * 256,
                                p.cache.row_bytes % 16 == 0);
    }
}

template <int FMT, int HD, typename T>
__global__ void __launch_bounds__(MOVE_WARPS * 32) kv_read_kernel(const MoveParams p) {
    __shared__ __align__(16) uint8_t stage_all[FMT == YUUKA_KV_Q8_0 ? MOVE_WARPS * MOVE_CHUNKS * Q8_CHUNK : 16];
    pdl_entry();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const MoveUnit u(p);
    if (u.chunks == 0) return;
    const int slot = move_slot(p, u.r);
    if (slot == -1) return;
    uint8_t * row = (u.is_v ? p.cache.v : p.cache.k) + (int64_t)max(slot, 0) * p.cache.row_bytes;
    // loads of all chunks first, then the values
    Eight<typename std::conditional<FMT == YUUKA_KV_F32, float, __half>::type> x[MOVE_CHUNKS];  // (F8: half of one)
    float d[MOVE_CHUNKS];
    if constexpr (FMT == YUUKA_KV_Q8_0) {
        if (slot >= 0) {
#pragma unroll
            for (int c = 0; c < MOVE_CHUNKS; c++)
                if (c < u.chunks)
                    move_q8_chunk<false>(stage_all + (warp * MOVE_CHUNKS + c) * Q8_CHUNK, row + (u.first / 256 + c) * Q8_CHUNK,
                                         p.kv_dim - u.first - c * 256, p.cache.row_bytes % 16 == 0);
            __syncwarp();
        }
    } else {
#pragma unroll
        for (int c = 0; c < MOVE_CHUNKS; c++) {
            const int first = u.first + c * 256 + lane * 8;
            if (slot < 0 || first >= p.kv_dim) continue;
            if constexpr (FMT == YUUKA_KV_F32) x[c].load(row + 4 * first);
            else if constexpr (FMT == YUUKA_KV_F16) x[c].load(row + 2 * first);
            else {
                const uint2 raw = __ldg(reinterpret_cast<const uint2 *>(row + first));
                x[c].raw[0].x = raw.x;
                x[c].raw[0].y = raw.y;
                d[c] = __ldg(reinterpret_cast<const float *>(row + p.kv_dim) + first / HD);
            }
        }
    }
    T * dst = reinterpret_cast<T *>(u.is_v ? p.v : p.k) + (int64_t)u.r * (u.is_v ? p.v_stride : p.k_stride) + u.first + lane * 8;
#pragma unroll
    for (int c = 0; c < MOVE_CHUNKS; c++) {
        if (u.first + c * 256 + lane * 8 >= p.kv_dim) break;
        float f[8];
        if constexpr (FMT == YUUKA_KV_Q8_0) {
            const uint16_t * blk = reinterpret_cast<const uint16_t *>(stage_all + (warp * MOVE_CHUNKS + c) * Q8_CHUNK + (lane >> 2) * 34);
            const float s = __half2float(__ushort_as_half(blk[0]));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint16_t q = blk[1 + (lane & 3) * 4 + i];
                f[2 * i] = s * (float)(int8_t)(q & 0xff);
                f[2 * i + 1] = s * (float)(int8_t)(q >> 8);
            }
        } else if constexpr (FMT == YUUKA_KV_F8) {
            const uint32_t raw[2] = {x[c].raw[0].x, x[c].raw[0].y};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const __nv_fp8x2_storage_t e = (__nv_fp8x2_storage_t)(raw[i >> 1] >> (16 * (i & 1)));
                const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(e, __NV_E4M3)));
                f[2 * i] = d[c] * v.x;
                f[2 * i + 1] = d[c] * v.y;
            }
        } else {
            x[c].get(f);
        }
        if (slot < 0)
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = __uint_as_float(0x7fffffffu);
        store8(dst + c * 256, f);
    }
}

template <int FMT, int HD, typename T>
static void launch_move_as(yuuka_stream * stream, const MoveParams & p, bool write) {
    const int64_t grid = ((int64_t)p.rows * 2 * p.groups + MOVE_WARPS - 1) / MOVE_WARPS;
    launch_k(write ? kv_write_kernel<FMT, HD, T> : kv_read_kernel<FMT, HD, T>, (unsigned)grid, MOVE_WARPS * 32, 0, stream->s, p);
}
template <int FMT, typename T> static void launch_move_format(yuuka_stream * stream, const MoveParams & p, bool write, int head_dim) {
    if constexpr (FMT == YUUKA_KV_F8) {  // (the other formats know no heads)
        if (head_dim == 64) return launch_move_as<FMT, 64, T>(stream, p, write);
        if (head_dim == 256) return launch_move_as<FMT, 256, T>(stream, p, write);
    }
    launch_move_as<FMT, 128, T>(stream, p, write);
}
template <typename T> static void launch_move(yuuka_stream * stream, const MoveParams & p, bool write, int head_dim) {
    switch (p.cache.format) {
    case YUUKA_KV_F32: return launch_move_format<YUUKA_KV_F32, T>(stream, p, write, head_dim);
    case YUUKA_KV_F16: return launch_move_format<YUUKA_KV_F16, T>(stream, p, write, head_dim);
    case YUUKA_KV_Q8_0: return launch_move_format<YUUKA_KV_Q8_0, T>(stream, p, write, head_dim);
    default: return launch_move_format<YUUKA_KV_F8, T>(stream, p, write, head_dim);
    }
}

static yuuka_status move_rows(const char * op, bool write, yuuka_stream * stream, const yuuka_kv_cache * cache, const yuuka_kv_rows * rows,
                              yuuka_event * completion) {
    return guard([&] {
        YK_REQUIRE(stream && cache && rows, YUUKA_ERR_INVALID_ARGUMENT, "%s: null argument", op);
        const yuuka_device * dev = stream->dev;
        MoveParams p;
        p.cache = check_cache(op, cache, dev);
        YK_REQUIRE(rows->rows >= 1 && rows->rows <= INT_MAX, YUUKA_ERR_INVALID_ARGUMENT, "%s: %llu rows", op, (unsigned long long)rows->rows);
        YK_REQUIRE(rows->dtype == YUUKA_DTYPE_F32 || rows->dtype == YUUKA_DTYPE_F16 || rows->dtype == YUUKA_DTYPE_BF16, YUUKA_ERR_UNSUPPORTED,
                   "%s: dtype %u is not F32, F16 or BF16", op, rows->dtype);
        const uint64_t size = rows->dtype == YUUKA_DTYPE_F32 ? 4 : 2, dim = (uint64_t)cache->kv_heads * (uint64_t)cache->head_dim;
        const uint64_t ks = rows->k_stride ? rows->k_stride : dim, vs = rows->v_stride ? rows->v_stride : dim;
        YK_REQUIRE(ks >= dim && vs >= dim, YUUKA_ERR_INVALID_ARGUMENT, "%s: row stride below %llu elements", op, (unsigned long long)dim);
        // (beyond it strides in bytes would leave 64 bits)
        YK_REQUIRE(ks <= 1ull << 48 && vs <= 1ull << 48, YUUKA_ERR_INVALID_ARGUMENT, "%s: row stride range exceeds 2^48 elements", op);
        YK_REQUIRE(ks * size % 16 == 0 && vs * size % 16 == 0, YUUKA_ERR_INVALID_ARGUMENT, "%s: row strides must be multiples of 16 bytes", op);
        const uint64_t kb = span_bytes(rows->rows, ks, 1, 0, dim, size), vb = span_bytes(rows->rows, vs, 1, 0, dim, size);
        check_range(op, "k", rows->k, rows->k_offset, kb, 16, dev);
        check_range(op, "v", rows->v, rows->v_offset, vb, 16, dev);
        check_range(op, "pos", rows->pos, rows->pos_offset, 4 * rows->rows, 4, dev);
        if (rows->seq) check_range(op, "seq", rows->seq, rows->seq_offset, 4 * rows->rows, 4, dev);
        if (rows->status) check_range(op, "status", rows->status, rows->status_offset, 4, 4, dev);
        // what is written lies over nothing that is read
        const uint64_t pool = (uint64_t)p.cache.row_bytes * (uint64_t)cache->block_size * (uint64_t)cache->pool_blocks,
                       tb = 4ull * (uint64_t)cache->sequences * (uint64_t)cache->table_stride;
        struct Range {
            const char * name;
            const yuuka_buffer * buf;
            uint64_t offset, bytes;
        };
        const Range pools[2] = {{"the K pool", cache->k, cache->k_offset, pool}, {"the V pool", cache->v, cache->v_offset, pool}};
        const Range nums[2] = {{"k", rows->k, rows->k_offset, kb}, {"v", rows->v, rows->v_offset, vb}};
        const Range lists[3] = {{"the block table", cache->tables, cache->tables_offset, tb},
                                {"pos", rows->pos, rows->pos_offset, 4 * rows->rows},
                                {"seq", rows->seq, rows->seq_offset, 4 * rows->rows}};
        const Range status = {"status", rows->status, rows->status_offset, 4};
        auto apart = [&](const Range & a, const Range & b) { check_apart(op, a.name, a.buf, a.offset, a.bytes, b.name, b.buf, b.offset, b.bytes); };
        for (const Range & a : write ? pools : nums) {
            for (const Range & b : write ? nums : pools) apart(a, b);
            for (const Range & b : lists) apart(a, b);
            apart(a, status);
        }
        for (const Range & b : lists) apart(status, b);
        for (const Range & b : write ? nums : pools) apart(status, b);
        if (!write) {
            // (two strided arrays may lie side by side in one: the rows themselves must not meet)
            const uint64_t k0 = (uint64_t)(uintptr_t)rows->k->ptr + rows->k_offset, v0 = (uint64_t)(uintptr_t)rows->v->ptr + rows->v_offset;
            const uint64_t apart = v0 > k0 ? v0 - k0 : k0 - v0, stride = ks * size, row = dim * size;
            const bool interleaved = ks == vs && apart % stride >= row && apart % stride + row <= stride;
            if (!interleaved) check_apart(op, "k", rows->k, rows->k_offset, kb, "v", rows->v, rows->v_offset, vb);
        }
        p.k = (uint8_t *)rows->k->ptr + rows->k_offset;
        p.v = (uint8_t *)rows->v->ptr + rows->v_offset;
        p.k_stride = (int64_t)ks;
        p.v_stride = (int64_t)vs;
        p.pos = (const int32_t *)((const uint8_t *)rows->pos->ptr + rows->pos_offset);
        p.seq = rows->seq ? (const int32_t *)((const uint8_t *)rows->seq->ptr + rows->seq_offset) : nullptr;
        p.status = rows->status ? (int32_t *)((uint8_t *)rows->status->ptr + rows->status_offset) : nullptr;
        p.rows = (int)rows->rows;
        p.kv_dim = (int)dim;
        p.groups = (int)((dim + 256 * MOVE_CHUNKS - 1) / (256 * MOVE_CHUNKS));
        // (warps are counted in 32 bits)
        YK_REQUIRE(rows->rows * 2 * (uint64_t)p.groups < (1ull << 32) - MOVE_WARPS, YUUKA_ERR_UNSUPPORTED, "%s: %llu rows of %llu values", op,
                   (unsigned long long)rows->rows, (unsigned long long)dim);
        set_device(dev);
        if (rows->dtype == YUUKA_DTYPE_F32) launch_move<float>(stream, p, write, cache->head_dim);
        else if (rows->dtype == YUUKA_DTYPE_F16) launch_move<__half>(stream, p, write, cache->head_dim);
        else launch_move<__nv_bfloat16>(stream, p, write, cache->head_dim);
        record_completion(stream, completion);
    });
}

}  // namespace yk

extern "C" uint64_t yuuka_kv_row_bytes(int32_t format, int32_t kv_heads, int32_t head_dim) {
    return yk::kv_row_bytes(format, kv_heads, head_dim);
}

extern "C" yuuka_status yuuka_kv_write(yuuka_stream * stream, const yuuka_kv_cache * cache, const yuuka_kv_rows * rows,
                                       yuuka_event * completion) {
    return yk::move_rows("kv_write", true, stream, cache, rows, completion);
}

extern "C" yuuka_status yuuka_kv_read(yuuka_stream * stream, const yuuka_kv_cache * cache, const yuuka_kv_rows * rows,
                                      yuuka_event * completion) {
    return yk::move_rows("kv_read", false, stream, cache, rows, completion);
}
