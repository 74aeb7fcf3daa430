// More of what the cache calls refuse, and of their kernels' bounds, on the host: with the operands and the compiled-in entry
// points of cache_checks.cu.
#define main cache_checks_main
#include "cache_checks.cu"
#undef main

// Every join that a call's second kernel takes for its own lies in the partial sums, whatever another call has left in the list.
template <int FMT, int HD, int NT, bool WIDE> static void joins_stay_inside() {
    using namespace yk;
    using S = DecodeShape<FMT, HD, NT, WIDE>;
    DecodeParams p{};
    p.batch = 8;
    p.head_tiles = 1;
    p.warps = 148 * S::RESIDENT * S::W;
    for (int units : {1, 2, 3, 16, 40, 592, 1024}) {
        p.cache.kv_heads = units;
        bool inside = true, taken = units * 2 > p.warps;
        for (int last = 1; last < 2 * DEC_WARPS; last++) {
            if (!decode_join_sound(p, make_int4(7, units - 1, last - 1, last))) continue;
            taken = true;
            inside &= (((size_t)last * units + units - 1) * 2 + 1) * S::PART_FLOATS * sizeof(float) <= DEC_PARTIAL_BYTES;  // the heads' slot
            inside &= (((size_t)(last - 1) * units + units - 1) * 2 + 2) * S::PART_FLOATS * sizeof(float) <= DEC_PARTIAL_BYTES;
        }
        const int teams = p.warps / units;
        char name[96];
        snprintf(name, sizeof name, "joins of format %d, heads of %d, %d columns, %d units", FMT, HD, S::COLS, units);
        expect(inside && taken && !decode_join_sound(p, make_int4(7, units - 1, 0, teams)) && !decode_join_sound(p, make_int4(7, units, 0, 1)) &&
                   !decode_join_sound(p, make_int4(8, 0, 0, 1)) && !decode_join_sound(p, make_int4(0, 0, -1, 1)) && !decode_join_sound(p, make_int4(0, 0, 1, 1)) &&
                   (teams < 2 || decode_join_sound(p, make_int4(0, 0, 0, teams - 1))),
               name);
    }
}
template <int FMT, bool WIDE> static void joins_of_format() {
    joins_stay_inside<FMT, 64, 1, WIDE>();
    joins_stay_inside<FMT, 128, 1, WIDE>();
    joins_stay_inside<FMT, 256, 1, WIDE>();
    if constexpr (FMT != YUUKA_KV_F32) {
        joins_stay_inside<FMT, 64, 2, WIDE>();
        joins_stay_inside<FMT, 128, 2, WIDE>();
        joins_stay_inside<FMT, 256, 2, WIDE>();
    }
}

int main() {
    using namespace yk;
    constexpr int WRITE = 1, READ = 2, MOVE = 3, ATTEND = 4;
    const yuuka_status INVALID = YUUKA_ERR_INVALID_ARGUMENT;
    (void)WRITE, (void)READ;
    int devices = 0;

    // A single row has no second one for a stride to reach: its byte stride may wrap to zero all the same
    for (int power : {49, 61, 62, 63})
        refuses("one row, a stride beyond 64 bits in bytes", INVALID, "row stride range exceeds", [=](World & w) {
            w.rows.rows = 1;
            w.rows.k_stride = w.rows.v_stride = 1ull << power;
            return MOVE;
        });
    refuses("one row, the largest stride", INVALID, "row stride range exceeds", [](World & w) {
        w.rows.rows = 1;
        w.rows.v_stride = ~0ull - 127;
        return MOVE;
    });

    // a scale whose product with log2 e is no f32: all scores would be infinite or NaN
    for (float scale : {2.4e38f, -3.4e38f, NAN})
        refuses("scale beyond its base-2 form", INVALID, "finite", [=](World & w) { w.args.scale = scale; return ATTEND; });

    // 1.5e9 tiles of 65536 rows, whatever the number of heads (nothing but the device is missing; nothing is launched with one)
    if (cudaGetDeviceCount(&devices) != cudaSuccess || devices == 0)
        refuses("tables of many keys and heads", YUUKA_ERR_DEVICE, "cudaSetDevice", [](World & w) {
            auto apart = [&](int i) {
                yuuka_buffer * b = w.buffer(0, 0);
                b->ptr = (void *)(uintptr_t)((1ull << 50) + ((uint64_t)i << 42));
                b->bytes = 1ull << 41;
                return b;
            };
            w.cache.block_size = 122880;
            w.cache.pool_blocks = 1;
            w.cache.k = apart(0);
            w.cache.v = apart(1);
            w.args.heads = 64;
            w.args.batch = 65536;
            w.args.q = apart(2);
            w.args.out = apart(3);
            w.args.gate = apart(4);
            w.args.lse = apart(5);
            w.args.lens = apart(6);
            w.args.seq_ids = apart(7);
            return ATTEND;
        });

    joins_of_format<YUUKA_KV_F32, true>();
    joins_of_format<YUUKA_KV_F32, false>();
    joins_of_format<YUUKA_KV_F16, true>();
    joins_of_format<YUUKA_KV_F16, false>();
    joins_of_format<YUUKA_KV_Q8_0, true>();
    joins_of_format<YUUKA_KV_Q8_0, false>();
    joins_of_format<YUUKA_KV_F8, true>();
    joins_of_format<YUUKA_KV_F8, false>();

    expect(launches == 0, "nothing was launched");
    printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures != 0;
}
