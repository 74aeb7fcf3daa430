// What the cache calls refuse, and where the kernels' own lookups send ids that are out of range, on the host: the entry
// points and the lookup functions are compiled as they are, buffers are host memory, and no kernel runs (the launches of the
// attention are replaced). A call that passes every check ends at the first CUDA call.
#include "attention_decode.cu"
#include "bridge.cu"
#include "kv_cache.cu"

#include <cstdio>
#include <cstring>
#include <vector>

namespace yk {
static int launches = 0;
void launch_decode_f32(cudaStream_t, const DecodeParams &, int, int, int) { launches++; }
void launch_decode_f16(cudaStream_t, const DecodeParams &, int, int, int) { launches++; }
void launch_decode_q8_0(cudaStream_t, const DecodeParams &, int, int, int) { launches++; }
void launch_decode_f8(cudaStream_t, const DecodeParams &, int, int, int) { launches++; }
}  // namespace yk

static int failures = 0;
static void expect(bool ok, const char * what) {
    if (!ok) {
        printf("FAIL %s (%s)\n", what, yuuka_last_error());
        failures++;
    }
}

struct World {
    alignas(256) uint8_t memory[1 << 20];
    yuuka_device dev, other;
    yuuka_stream stream;
    yuuka_attention_scratch scratch;
    std::vector<yuuka_buffer> buffers;
    yuuka_kv_cache cache{};
    yuuka_kv_rows rows{};
    yuuka_attention_decode_args args{};
    yuuka_buffer * buffer(size_t at, size_t bytes) {
        yuuka_buffer b;
        b.dev = &dev;
        b.ptr = memory + at;
        b.bytes = bytes;
        b.view = true;
        buffers.push_back(b);
        return &buffers.back();
    }
    World() {
        buffers.reserve(32);
        dev.index = 0;
        dev.sm_count = 148;
        other.index = 1;
        stream.dev = &dev;
        scratch.dev = &dev;
        scratch.memory = memory + (900 << 10);
        // two sequences of three blocks of four rows, two KV heads of 64, f16: 256 bytes a row
        cache.k = buffer(0, 6 * 4 * 256);
        cache.v = buffer(8192, 6 * 4 * 256);
        cache.tables = buffer(16384, 2 * 3 * 4);
        cache.format = YUUKA_KV_F16;
        cache.kv_heads = 2;
        cache.head_dim = 64;
        cache.block_size = 4;
        cache.pool_blocks = 6;
        cache.sequences = 2;
        cache.table_stride = 3;
        rows.k = buffer(32768, 5 * 128 * 4);
        rows.v = buffer(40960, 5 * 128 * 4);
        rows.pos = buffer(49152, 20);
        rows.seq = buffer(49408, 20);
        rows.status = buffer(49664, 4);
        rows.rows = 5;
        rows.dtype = YUUKA_DTYPE_F32;
        args.q = buffer(65536, 2 * 8 * 64 * 4);
        args.out = buffer(73728, 2 * 8 * 64 * 4);
        args.gate = buffer(81920, 2 * 8 * 64 * 4);
        args.lse = buffer(90112, 2 * 8 * 4);
        args.lens = buffer(98304, 8);
        args.seq_ids = buffer(98560, 8);
        args.status = buffer(98816, 4);
        args.dtype = YUUKA_DTYPE_F32;
        args.batch = 2;
        args.heads = 8;
    }
};

template <typename F> static void refuses(const char * what, yuuka_status want, const char * words, F change) {
    // every call that the change concerns answers `want`, with these words in its message
    for (int call = 0; call < 3; call++) {
        World * w = new World();
        const int mask = change(*w);
        if (mask >> call & 1) {
            const yuuka_status got = call == 0   ? yuuka_kv_write(&w->stream, &w->cache, &w->rows, nullptr)
                                     : call == 1 ? yuuka_kv_read(&w->stream, &w->cache, &w->rows, nullptr)
                                                 : yuuka_attention_decode(&w->stream, &w->scratch, &w->cache, &w->args, nullptr);
            char name[128];
            snprintf(name, sizeof name, "%s, call %d, status %d", what, call, (int)got);
            expect(got == want && strstr(yuuka_last_error(), words), name);
        }
        delete w;
    }
}

int main() {
    using namespace yk;
    constexpr int WRITE = 1, READ = 2, MOVE = 3, ATTEND = 4, ALL = 7;
    const yuuka_status INVALID = YUUKA_ERR_INVALID_ARGUMENT, UNSUPPORTED = YUUKA_ERR_UNSUPPORTED;

    // as they stand, the calls pass their checks: without a device the next thing fails, with one it is the launch of a kernel
    // on host memory, which is not done here
    int devices = 0;
    if (cudaGetDeviceCount(&devices) != cudaSuccess || devices == 0)
        refuses("valid calls", YUUKA_ERR_DEVICE, "cudaSetDevice", [](World &) { return ALL; });

    refuses("format", INVALID, "KV format", [](World & w) { w.cache.format = 4; return ALL; });
    refuses("no KV heads", INVALID, "KV heads", [](World & w) { w.cache.kv_heads = 0; return ALL; });
    refuses("head dimension", UNSUPPORTED, "head_dim", [](World & w) { w.cache.head_dim = 96; return ALL; });
    refuses("block size", INVALID, "blocks of", [](World & w) { w.cache.block_size = 0; return ALL; });
    refuses("pool rows", INVALID, "blocks of", [](World & w) { w.cache.block_size = w.cache.pool_blocks = 1 << 16; return ALL; });
    refuses("no tables", INVALID, "block tables", [](World & w) { w.cache.table_stride = 0; return ALL; });
    refuses("K pool too small", INVALID, "K pool range", [](World & w) { w.cache.k->bytes--; return ALL; });
    refuses("V pool too small", INVALID, "V pool range", [](World & w) { w.cache.v_offset = 16; return ALL; });
    refuses("V pool misaligned", INVALID, "multiple of 16", [](World & w) { w.cache.v->bytes += 64; w.cache.v_offset = 8; return ALL; });
    refuses("pools overlap", INVALID, "lies over", [](World & w) { w.cache.v->ptr = w.memory + 4096; return ALL; });
    refuses("table too small", INVALID, "block table range", [](World & w) { w.cache.sequences = 3; return ALL; });
    refuses("null pool", INVALID, "K pool is null", [](World & w) { w.cache.k = nullptr; return ALL; });
    refuses("another device", INVALID, "on device 1", [](World & w) { w.cache.k->dev = &w.other; return ALL; });
    refuses("no rows", INVALID, "0 rows", [](World & w) { w.rows.rows = 0; return MOVE; });
    refuses("too many rows", INVALID, "range exceeds", [](World & w) { w.rows.rows = 6; return MOVE; });
    refuses("rows past 31 bits", INVALID, "rows", [](World & w) { w.rows.rows = 1ull << 31; return MOVE; });
    refuses("row type", UNSUPPORTED, "dtype", [](World & w) { w.rows.dtype = YUUKA_DTYPE_Q8_0; return MOVE; });
    refuses("row stride too small", INVALID, "row stride", [](World & w) { w.rows.k_stride = 124; return MOVE; });
    refuses("row stride misaligned", INVALID, "multiples of 16", [](World & w) { w.rows.rows = 1; w.rows.v_stride = 130; return MOVE; });
    refuses("row stride out of range", INVALID, "range exceeds", [](World & w) { w.rows.v_stride = 1ull << 60; return MOVE; });
    refuses("rows over the pool", INVALID, "lies over", [](World & w) { w.rows.k->ptr = w.memory + 1024; return MOVE; });
    refuses("read: k over v", INVALID, "lies over", [](World & w) { w.rows.v->ptr = w.memory + 32768 + 256; return READ; });
    refuses("read: rows over pos", INVALID, "lies over", [](World & w) { w.rows.pos = w.buffer(32768, 20); return READ; });
    refuses("no positions", INVALID, "pos is null", [](World & w) { w.rows.pos = nullptr; return MOVE; });
    refuses("seq too small", INVALID, "seq range", [](World & w) { w.rows.seq = w.buffer(49408, 16); return MOVE; });
    refuses("q type", UNSUPPORTED, "dtype", [](World & w) { w.args.dtype = YUUKA_DTYPE_Q8_0; return ATTEND; });
    refuses("no batch", INVALID, "batch 0", [](World & w) { w.args.batch = 0; return ATTEND; });
    refuses("heads", INVALID, "heads", [](World & w) { w.args.heads = 7; return ATTEND; });
    refuses("batch beyond sequences", INVALID, "without sequence ids", [](World & w) {
        w.args.seq_ids = nullptr;
        w.args.batch = 3;
        return ATTEND;
    });
    refuses("window", INVALID, "window", [](World & w) { w.args.window = -1; return ATTEND; });
    refuses("scale", INVALID, "finite", [](World & w) { w.args.scale = INFINITY; return ATTEND; });
    refuses("q too small", INVALID, "q range", [](World & w) { w.args.q_head_stride = 128; return ATTEND; });
    refuses("q misaligned", INVALID, "multiple of 16", [](World & w) { w.args.batch = 1; w.args.q_offset = 4; return ATTEND; });
    refuses("q stride misaligned", INVALID, "multiples of 16", [](World & w) { w.args.batch = 1; w.args.q_head_stride = 66; return ATTEND; });
    refuses("q stride out of range", INVALID, "stride", [](World & w) { w.args.q_head_stride = ~0ull; return ATTEND; });
    refuses("out rows overlap", INVALID, "overlap", [](World & w) { w.args.out_row_stride = 64; return ATTEND; });
    refuses("out over q", INVALID, "out lies over q", [](World & w) { w.args.out = (yuuka_buffer *)w.args.q; return ATTEND; });
    refuses("out over a pool", INVALID, "lies over", [](World & w) { w.args.out->ptr = w.cache.v->ptr; return ATTEND; });
    refuses("lse over lens", INVALID, "lies over", [](World & w) { w.args.lse->ptr = w.memory + 98304 - 32; return ATTEND; });
    // status bits are or-ed into memory that the call reads nowhere else
    refuses("status over pos", INVALID, "status lies over pos", [](World & w) { w.rows.status = (yuuka_buffer *)w.rows.pos; return MOVE; });
    refuses("status over seq", INVALID, "status lies over seq", [](World & w) { w.rows.status->ptr = w.memory + 49408 + 16; return MOVE; });
    refuses("status over the table", INVALID, "status lies over the block table", [](World & w) {
        w.rows.status = w.args.status = (yuuka_buffer *)w.cache.tables;
        return ALL;
    });
    refuses("status over rows that are read", INVALID, "status lies over k", [](World & w) { w.rows.status->ptr = w.memory + 32768 + 64; return WRITE; });
    refuses("status over a pool that is read", INVALID, "status lies over the V pool", [](World & w) {
        w.rows.status->ptr = w.args.status->ptr = w.memory + 8192;
        return READ | ATTEND;
    });
    refuses("status over lens", INVALID, "status lies over lens", [](World & w) { w.args.status->ptr = w.memory + 98304 + 4; return ATTEND; });
    refuses("status over q", INVALID, "status lies over q", [](World & w) { w.args.status->ptr = w.memory + 65536; return ATTEND; });
    refuses("status over out", INVALID, "out lies over status", [](World & w) { w.args.status->ptr = w.memory + 73728 + 4; return ATTEND; });
    refuses("no lengths", INVALID, "lens is null", [](World & w) { w.args.lens = nullptr; return ATTEND; });
    refuses("scratch of another device", INVALID, "scratch is on device 1", [](World & w) { w.scratch.dev = &w.other; return ATTEND; });
    refuses("too many keys", UNSUPPORTED, "too many", [](World & w) {
        // (buffers of these sizes nowhere: the call ends before it uses them)
        auto apart = [&](int i) {
            yuuka_buffer * b = w.buffer(0, 0);
            b->ptr = (void *)(uintptr_t)((1ull << 50) + ((uint64_t)i << 42));
            b->bytes = 1ull << 41;
            return b;
        };
        w.cache.block_size = 1 << 28;
        w.cache.pool_blocks = 1;
        w.cache.k = apart(0);
        w.cache.v = apart(1);
        w.args.heads = 2;
        w.args.batch = 65536;
        w.args.q = apart(2);
        w.args.out = apart(3);
        w.args.gate = apart(4);
        w.args.lse = apart(5);
        w.args.lens = apart(6);
        w.args.seq_ids = apart(7);
        return ATTEND;
    });
    expect(yuuka_kv_write(nullptr, nullptr, nullptr, nullptr) == INVALID, "null write");
    expect(yuuka_kv_read(nullptr, nullptr, nullptr, nullptr) == INVALID, "null read");
    expect(yuuka_attention_decode(nullptr, nullptr, nullptr, nullptr, nullptr) == INVALID, "null attention");
    expect(launches == 0, "nothing was launched");

    // lookups
    World * w = new World();
    PagedCache c = check_cache("lookup", &w->cache, &w->dev);
    int32_t * tables = (int32_t *)(w->memory + 16384);
    const int32_t ids[6] = {5, 0, 3, -1, 6, 2};
    memcpy(tables, ids, sizeof ids);
    int bad = 0;
    expect(c.capacity == 12 && c.shift == 2, "capacity");
    expect(kv_token_slot(c, 0, 0, bad) == 20 && !bad, "first row");
    expect(kv_token_slot(c, 0, 11, bad) == 15 && !bad, "last row");
    expect(kv_token_slot(c, 1, 11, bad) == 11 && !bad, "a table's last block");
    expect(kv_token_slot(c, 0, 12, bad) == -2 && bad == YUUKA_KV_STATUS_POSITION, "a position beyond the table");
    expect(kv_token_slot(c, 0, INT_MAX, bad) == -2 && bad == YUUKA_KV_STATUS_POSITION, "the largest position");
    expect(kv_token_slot(c, 1, 3, bad) == -2 && bad == YUUKA_KV_STATUS_BLOCK, "a block below the pool");
    expect(kv_token_slot(c, 1, 4, bad) == -2 && bad == YUUKA_KV_STATUS_BLOCK, "a block beyond the pool");
    expect(kv_token_slot(c, 2, 0, bad) == -2 && bad == YUUKA_KV_STATUS_SEQUENCE, "a sequence beyond the tables");
    expect(kv_token_slot(c, -1, 0, bad) == -2 && bad == YUUKA_KV_STATUS_SEQUENCE, "a sequence below the tables");
    expect(kv_token_slot(c, 7, -1, bad) == -1 && !bad, "no token");
    c.shift = -1;  // (a block size that is no power of two divides)
    c.block_size = 3;
    expect(kv_token_slot(c, 0, 7, bad) == 10 && !bad, "a block of three rows");

    DecodeParams p{};
    p.cache = check_cache("lookup", &w->cache, &w->dev);
    int32_t lens[6] = {0, 12, 13, -1, 5, 1}, seqs[6] = {0, 1, 0, 1, 2, -1};
    p.lens = lens;
    p.seq_ids = seqs;
    p.batch = 6;
    DecodeSpan s = decode_span(p, 0, 16, bad);
    expect(s.tiles == 1 && s.end == 0 && s.seq == 0 && !bad, "a row without keys has a tile");
    s = decode_span(p, 1, 16, bad);
    expect(s.tiles == 1 && s.first == 0 && s.end == 12 && s.seq == 1 && !bad, "a full table");
    s = decode_span(p, 2, 16, bad);
    expect(s.tiles == 1 && s.end == 0 && s.seq == -1 && bad == YUUKA_KV_STATUS_POSITION, "a length beyond the table");
    s = decode_span(p, 3, 16, bad);
    expect(s.tiles == 1 && s.end == 0 && s.seq == -1 && bad == YUUKA_KV_STATUS_POSITION, "a length below zero");
    s = decode_span(p, 4, 16, bad);
    expect(s.tiles == 1 && s.seq == -1 && bad == YUUKA_KV_STATUS_SEQUENCE, "a sequence beyond the tables");
    s = decode_span(p, 5, 16, bad);
    expect(s.tiles == 1 && s.seq == -1 && bad == YUUKA_KV_STATUS_SEQUENCE, "a sequence below the tables");
    p.window = 5;
    s = decode_span(p, 1, 16, bad);
    expect(s.tiles == 1 && s.first == 7 && s.end == 12, "a window");
    p.cache.capacity = INT_MAX;
    lens[1] = INT_MAX;
    p.window = 0;
    s = decode_span(p, 1, 16, bad);
    expect(s.tiles == 1 << 27 && s.end == INT_MAX && !bad, "the longest sequence");

    expect(yuuka_kv_row_bytes(YUUKA_KV_F32, 3, 64) == 768 && yuuka_kv_row_bytes(YUUKA_KV_F16, 3, 64) == 384 &&
               yuuka_kv_row_bytes(YUUKA_KV_Q8_0, 3, 64) == 204 && yuuka_kv_row_bytes(YUUKA_KV_F8, 3, 64) == 208 &&
               yuuka_kv_row_bytes(YUUKA_KV_F8, 4, 256) == 1040 && yuuka_kv_row_bytes(4, 1, 64) == 0 && yuuka_kv_row_bytes(0, 1, 32) == 0,
           "row bytes");
    delete w;
    printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures != 0;
}
