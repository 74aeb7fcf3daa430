// A paged key-value cache in buffers of the caller: what yuuka_kv_write, yuuka_kv_read and yuuka_attention_decode share.
#pragma once

#include "common.cuh"

namespace yk {

// Pools [pool_blocks][block_size][row_bytes], addressed by position through block tables (kv_pool.go:117-134,
// memory/memory.go:253-266).
struct PagedCache {
    uint8_t * k;
    uint8_t * v;
    const int32_t * tables;  // [sequences][table_stride]
    int64_t row_bytes;
    int format, kv_heads, block_size, pool_blocks, sequences, table_stride;
    int shift;     // log2 of the block size, or -1
    int capacity;  // positions that a block table can map
};

constexpr int KV_BAD_BLOCK = YUUKA_KV_STATUS_BLOCK, KV_BAD_SEQUENCE = YUUKA_KV_STATUS_SEQUENCE,
              KV_BAD_POSITION = YUUKA_KV_STATUS_POSITION;

// Bytes of one row, 0 for a format or shape without a form.
uint64_t kv_row_bytes(int32_t format, int32_t kv_heads, int32_t head_dim);
// Checks numbers, ranges and overlaps of a cache and gives the kernels' form of it; throws. The second: the numbers alone.
PagedCache check_cache(const char * op, const yuuka_kv_cache * cache, const yuuka_device * dev);
void check_geometry(const char * op, const yuuka_kv_cache * cache);

// Bytes that a strided [rows][heads][dim] array spans, or UINT64_MAX where that passes 2^62.
uint64_t span_bytes(uint64_t rows, uint64_t row_stride, uint64_t heads, uint64_t head_stride, uint64_t dim, uint64_t size);
// Checks that [offset, offset + bytes) lies in the buffer, on the device, and starts at a multiple of `align` bytes.
void check_range(const char * op, const char * what, const yuuka_buffer * buf, uint64_t offset, uint64_t bytes, uint64_t align,
                 const yuuka_device * dev);
// Refuses an output that lies over another operand.
void check_apart(const char * op, const char * a_name, const yuuka_buffer * a, uint64_t a_offset, uint64_t a_bytes, const char * b_name,
                 const yuuka_buffer * b, uint64_t b_offset, uint64_t b_bytes);

#ifdef __CUDACC__
__host__ __device__ __forceinline__ int32_t kv_load(const int32_t * p) {
#ifdef __CUDA_ARCH__
    return __ldg(p);
#else
    return *p;
#endif
}
// Row of the pools that holds position pos of a sequence whose block table this is: the caller has checked
// 0 <= pos < capacity. -2 where the table names a block that the pools do not have.
__host__ __device__ __forceinline__ int kv_slot(const PagedCache & c, const int32_t * table, int pos) {
    const int page = c.shift >= 0 ? pos >> c.shift : pos / c.block_size;
    const int block = kv_load(table + page);
    return (unsigned)block < (unsigned)c.pool_blocks ? block * c.block_size + (pos - page * c.block_size) : -2;
}
// The same for position pos of sequence seq, all of it read from the device: -1 without a token (pos < 0), -2 with the status
// bit in `bad` where something is out of range.
__host__ __device__ __forceinline__ int kv_token_slot(const PagedCache & c, int seq, int pos, int & bad) {
    bad = 0;
    if (pos < 0) return -1;
    if ((unsigned)seq >= (unsigned)c.sequences) bad = KV_BAD_SEQUENCE;
    else if (pos >= c.capacity) bad = KV_BAD_POSITION;
    if (bad) return -2;
    const int slot = kv_slot(c, c.tables + (int64_t)seq * c.table_stride, pos);
    if (slot < 0) bad = KV_BAD_BLOCK;
    return slot;
}
#endif

}  // namespace yk
