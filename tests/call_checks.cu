// More of what the cache calls refuse, and of their kernels' bounds, on the host: with the operands and the compiled-in entry
// points of cache_checks.cu.
#define main cache_checks_main
#include "cache_checks.cu"
#undef main

int main() {
    using namespace yk;
    constexpr int WRITE = 1, READ = 2, MOVE = 3, ATTEND = 4;
    const yuuka_status INVALID = YUUKA_ERR_INVALID_ARGUMENT;
    (void)WRITE, (void)READ, (void)ATTEND;

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

    expect(launches == 0, "nothing was launched");
    printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures != 0;
}
