// yuuka_attention_decode: checks of arguments, scratch, choice of the kernel.
#include <algorithm>
#include <climits>
#include <cmath>

#include "attention_decode.cuh"

struct yuuka_attention_scratch {
    yuuka_device * dev = nullptr;
    uint8_t * memory = nullptr;
};

namespace yk {

// the scratch memory: counters, joins of both lists, runs to be done again, partials
constexpr size_t DEC_JOINS_AT = (DEC_COUNTERS * sizeof(int) + 255) / 256 * 256, DEC_FAR_AT = DEC_JOINS_AT + 2 * DEC_WARPS * sizeof(int4),
                 DEC_PARTIAL_AT = DEC_FAR_AT + DEC_FAR_MOST * sizeof(int2);

// rows and heads of an output: either all heads of a row behind one another or all rows of a head
static bool strides_disjoint(uint64_t rows, uint64_t row, uint64_t heads, uint64_t head, uint64_t dim) {
    const unsigned __int128 r = row, h = head;
    return (h >= dim && r >= (heads - 1) * h + dim) || (r >= dim && h >= (rows - 1) * r + dim);
}

}  // namespace yk

extern "C" yuuka_status yuuka_attention_scratch_create(yuuka_device * dev, yuuka_attention_scratch ** out) {
    using namespace yk;
    return guard([&] {
        YK_REQUIRE(out, YUUKA_ERR_INVALID_ARGUMENT, "attention_scratch_create: null argument");
        *out = nullptr;
        YK_REQUIRE(dev, YUUKA_ERR_INVALID_ARGUMENT, "attention_scratch_create: null argument");
        set_device(dev);
        void * ptr = nullptr;
        const size_t bytes = DEC_PARTIAL_AT + DEC_PARTIAL_BYTES;
        const cudaError_t err = cudaMalloc(&ptr, bytes);
        if (err != cudaSuccess) {
            cudaGetLastError();
            YK_REQUIRE(false, YUUKA_ERR_ALLOCATION, "cudaMalloc(%llu) failed: %s", (unsigned long long)bytes, cudaGetErrorString(err));
        }
        auto * s = new (std::nothrow) yuuka_attention_scratch();
        const cudaError_t zeroed = s ? cudaMemset(ptr, 0, DEC_JOINS_AT) : cudaSuccess;
        const cudaError_t waited = s && zeroed == cudaSuccess ? cudaDeviceSynchronize() : zeroed;
        if (!s || waited != cudaSuccess) {
            cudaFree(ptr);
            delete s;
            if (!s) throw std::bad_alloc();
            YK_CUDA(waited);
        }
        s->dev = dev;
        s->memory = (uint8_t *)ptr;
        *out = s;
    });
}

extern "C" void yuuka_attention_scratch_destroy(yuuka_attention_scratch * scratch) {
    if (!scratch) return;
    if (scratch->memory) {
        cudaSetDevice(scratch->dev->index);
        cudaFree(scratch->memory);
    }
    delete scratch;
}

extern "C" yuuka_status yuuka_attention_decode(yuuka_stream * stream, yuuka_attention_scratch * scratch, const yuuka_kv_cache * cache,
                                               const yuuka_attention_decode_args * a, yuuka_event * completion) {
    using namespace yk;
    return guard([&] {
        const char * op = "attention_decode";
        YK_REQUIRE(stream && scratch && cache && a, YUUKA_ERR_INVALID_ARGUMENT, "%s: null argument", op);
        const yuuka_device * dev = stream->dev;
        YK_REQUIRE(scratch->dev->index == dev->index, YUUKA_ERR_INVALID_ARGUMENT, "%s: the scratch is on device %d, the stream on device %d", op,
                   scratch->dev->index, dev->index);
        DecodeParams p;
        p.cache = check_cache(op, cache, dev);
        YK_REQUIRE(a->dtype == YUUKA_DTYPE_F32 || a->dtype == YUUKA_DTYPE_F16 || a->dtype == YUUKA_DTYPE_BF16, YUUKA_ERR_UNSUPPORTED,
                   "%s: dtype %u is not F32, F16 or BF16", op, a->dtype);
        YK_REQUIRE(a->batch >= 1 && a->batch <= 65536, YUUKA_ERR_INVALID_ARGUMENT, "%s: batch %d is not 1..65536", op, a->batch);
        YK_REQUIRE(a->heads >= 1 && a->heads <= 65536 && a->heads % cache->kv_heads == 0, YUUKA_ERR_INVALID_ARGUMENT,
                   "%s: %d heads are not a multiple of %d KV heads up to 65536", op, a->heads, cache->kv_heads);
        YK_REQUIRE(a->seq_ids || a->batch <= cache->sequences, YUUKA_ERR_INVALID_ARGUMENT, "%s: batch %d without sequence ids exceeds %d sequences", op,
                   a->batch, cache->sequences);
        YK_REQUIRE(a->window >= 0, YUUKA_ERR_INVALID_ARGUMENT, "%s: window %d", op, a->window);
        // (the kernel's factor, in base 2, is f32 as well)
        const double scale = a->scale != 0.0f ? (double)a->scale : 1.0 / std::sqrt((double)cache->head_dim);
        const float scale_log2 = (float)(scale * 1.4426950408889634);
        YK_REQUIRE(std::isfinite(scale_log2), YUUKA_ERR_INVALID_ARGUMENT, "%s: scale is not finite in f32 times log2 e", op);
        const uint64_t size = a->dtype == YUUKA_DTYPE_F32 ? 4 : 2, hd = (uint64_t)cache->head_dim, heads = (uint64_t)a->heads,
                       batch = (uint64_t)a->batch;
        const uint64_t qh = a->q_head_stride ? a->q_head_stride : hd, oh = a->out_head_stride ? a->out_head_stride : hd;
        YK_REQUIRE(qh <= UINT64_MAX / heads && oh <= UINT64_MAX / heads, YUUKA_ERR_INVALID_ARGUMENT, "%s: head stride out of range", op);
        const uint64_t qr = a->q_row_stride ? a->q_row_stride : heads * qh, orow = a->out_row_stride ? a->out_row_stride : heads * oh;
        for (const uint64_t s : {qh, qr, oh, orow})
            YK_REQUIRE(s <= (1ull << 48) && s * size % 16 == 0, YUUKA_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 16 bytes", op);
        YK_REQUIRE(strides_disjoint(batch, orow, heads, oh, hd), YUUKA_ERR_INVALID_ARGUMENT, "%s: rows or heads of out overlap", op);
        const uint64_t qb = span_bytes(batch, qr, heads, qh, hd, size), ob = span_bytes(batch, orow, heads, oh, hd, size);
        check_range(op, "q", a->q, a->q_offset, qb, 16, dev);
        check_range(op, "out", a->out, a->out_offset, ob, 16, dev);
        if (a->gate) check_range(op, "gate", a->gate, a->gate_offset, qb, 16, dev);
        if (a->lse) check_range(op, "lse", a->lse, a->lse_offset, 4 * batch * heads, 4, dev);
        check_range(op, "lens", a->lens, a->lens_offset, 4 * batch, 4, dev);
        if (a->seq_ids) check_range(op, "seq_ids", a->seq_ids, a->seq_ids_offset, 4 * batch, 4, dev);
        if (a->status) check_range(op, "status", a->status, a->status_offset, 4, 4, dev);
        const uint64_t pool = (uint64_t)p.cache.row_bytes * (uint64_t)cache->block_size * (uint64_t)cache->pool_blocks,
                       tb = 4ull * (uint64_t)cache->sequences * (uint64_t)cache->table_stride, lb = 4 * batch * heads;
        struct Range {
            const char * name;
            const yuuka_buffer * buf;
            uint64_t offset, bytes;
        };
        const Range outs[3] = {{"out", a->out, a->out_offset, ob}, {"lse", a->lse, a->lse_offset, lb}, {"status", a->status, a->status_offset, 4}};
        const Range ins[7] = {{"q", a->q, a->q_offset, qb},
                              {"gate", a->gate, a->gate_offset, qb},
                              {"lens", a->lens, a->lens_offset, 4 * batch},
                              {"seq_ids", a->seq_ids, a->seq_ids_offset, 4 * batch},
                              {"the K pool", cache->k, cache->k_offset, pool},
                              {"the V pool", cache->v, cache->v_offset, pool},
                              {"the block table", cache->tables, cache->tables_offset, tb}};
        for (const Range & x : outs)
            for (const Range & y : ins) check_apart(op, x.name, x.buf, x.offset, x.bytes, y.name, y.buf, y.offset, y.bytes);
        for (int i = 0; i < 3; i++)
            for (int j = 0; j < i; j++)
                check_apart(op, outs[j].name, outs[j].buf, outs[j].offset, outs[j].bytes, outs[i].name, outs[i].buf, outs[i].offset, outs[i].bytes);

        p.q = (const uint8_t *)a->q->ptr + a->q_offset;
        p.gate = a->gate ? (const uint8_t *)a->gate->ptr + a->gate_offset : nullptr;
        p.out = (uint8_t *)a->out->ptr + a->out_offset;
        p.lse = a->lse ? (float *)((uint8_t *)a->lse->ptr + a->lse_offset) : nullptr;
        p.lens = (const int32_t *)((const uint8_t *)a->lens->ptr + a->lens_offset);
        p.seq_ids = a->seq_ids ? (const int32_t *)((const uint8_t *)a->seq_ids->ptr + a->seq_ids_offset) : nullptr;
        p.status = a->status ? (int32_t *)((uint8_t *)a->status->ptr + a->status_offset) : nullptr;
        p.q_row = (int64_t)qr;
        p.q_head = (int64_t)qh;
        p.out_row = (int64_t)orow;
        p.out_head = (int64_t)oh;
        p.batch = a->batch;
        p.heads = a->heads;
        p.group = a->heads / cache->kv_heads;
        // Tiles of up to 16 query heads share one reading of the keys (8 over f32 pools, see launch_decode_f32)
        const int widest = cache->format == YUUKA_KV_F32 ? 8 : 16;
        p.head_tiles = (p.group + widest - 1) / widest;
        p.tile_heads = (p.group + p.head_tiles - 1) / p.head_tiles;
        const int cols = p.tile_heads <= 8 ? 8 : 16;
        p.window = a->window;
        p.dtype = (int)a->dtype;
        p.scale_log2 = scale_log2;
        p.counters = (int *)scratch->memory;
        p.joins = (int4 *)(scratch->memory + DEC_JOINS_AT);
        p.far = (int2 *)(scratch->memory + DEC_FAR_AT);
        p.partial = (float *)(scratch->memory + DEC_PARTIAL_AT);
        // a team's tiles, those of all rows at most, are counted in 31 bits
        const double tiles = (double)a->batch * (p.cache.capacity / 16 + 1.0);
        YK_REQUIRE(tiles < 2e9, YUUKA_ERR_UNSUPPORTED, "%s: %g tiles of keys are too many for one call", op, tiles);
        set_device(dev);
        switch (cache->format) {
        case YUUKA_KV_F32: launch_decode_f32(stream->s, p, cache->head_dim, cols, dev->sm_count); break;
        case YUUKA_KV_F16: launch_decode_f16(stream->s, p, cache->head_dim, cols, dev->sm_count); break;
        case YUUKA_KV_Q8_0: launch_decode_q8_0(stream->s, p, cache->head_dim, cols, dev->sm_count); break;
        default: launch_decode_f8(stream->s, p, cache->head_dim, cols, dev->sm_count); break;
        }
        record_completion(stream, completion);
    });
}
