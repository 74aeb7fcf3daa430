// Buffers of a foreign owner may begin at any byte: every call whose kernels read words refuses a range that does not start at
// a multiple of them. Handles are made by hand over host memory, and the calls end at the refusal, so no device is needed.
#include "common.cuh"

#include <cstdio>
#include <cstring>

static int failures = 0;
alignas(256) static uint8_t memory[1 << 20];
static yuuka_device device;

// 64 KB, `shift` bytes behind a multiple of 256
static yuuka_buffer * at(int slot, int shift) {
    static yuuka_buffer buffers[4];
    yuuka_buffer & b = buffers[slot];
    b.dev = &device;
    b.ptr = memory + (slot << 17) + shift;
    b.bytes = 1 << 16;
    b.view = true;
    return &b;
}
static void refused(yuuka_status got, const char * operand, const char * call, int shift) {
    const char * said = yuuka_last_error();
    const bool ok = got == YUUKA_ERR_INVALID_ARGUMENT && strstr(said, operand) && strstr(said, "does not start at a multiple");
    if (!ok) {
        printf("FAIL %s, %s %d bytes off: status %d, %s\n", call, operand, shift, (int)got, said);
        failures++;
    }
}

int main() {
    yuuka_stream stream;
    device.sm_count = 148;
    stream.dev = &device;
    const int shifts[] = {2, 4, 8, 12};
    for (int s : shifts) {
        auto gemm = [&](int w, int x, int out, uint32_t type, uint32_t flags) {
            return yuuka_gemm_quant(&stream, at(0, out), 0, at(1, x), 0, YUUKA_DTYPE_F32, at(2, w), 0, type, 256, 16, 4, YUUKA_GEMM_PATH_AUTO, flags, nullptr);
        };
        refused(gemm(s, 0, 0, YUUKA_DTYPE_Q4_K, YUUKA_GEMM_TILED), "the weights", "gemm_quant, tiled", s);
        for (uint32_t flags : {0u, YUUKA_GEMM_TILED}) {
            refused(gemm(0, s, 0, YUUKA_DTYPE_Q8_0, flags), "the activations", "gemm_quant", s);
            refused(gemm(0, 0, s, YUUKA_DTYPE_Q8_0, flags), "the output", "gemm_quant", s);
        }
        auto fixed = [&](int w, int x, int out) {
            return yuuka_gemm_quant_static(&stream, at(0, out), 0, at(1, x), 0, YUUKA_DTYPE_F32, at(2, w), 0, YUUKA_DTYPE_Q4_K, 256, 16, 4, YUUKA_GEMM_PATH_AUTO,
                                           YUUKA_GEMM_TILED, nullptr);
        };
        refused(fixed(s, 0, 0), "the weights", "gemm_quant_static", s);
        refused(fixed(0, s, 0), "the activations", "gemm_quant_static", s);
        refused(fixed(0, 0, s), "the output", "gemm_quant_static", s);
        refused(yuuka_weights_tile(&stream, at(0, s), 0, at(1, 1), 0, YUUKA_DTYPE_Q4_K, 16, 256, nullptr), "the destination", "weights_tile", s);
    }
    // offsets count from the address: a view 8 bytes off and an offset of 8 meet again, and the other way round
    refused(yuuka_gemm_quant(&stream, at(0, 0), 0, at(1, 8), 16, YUUKA_DTYPE_BF16, at(2, 0), 0, YUUKA_DTYPE_Q4_K, 256, 16, 1, YUUKA_GEMM_PATH_AUTO,
                             YUUKA_GEMM_TILED, nullptr),
            "the activations", "gemm_quant", 24);
    // rows in GGUF order: words of two bytes, of f32 four
    for (uint32_t type : {YUUKA_DTYPE_F16, YUUKA_DTYPE_Q8_0, YUUKA_DTYPE_Q6_K})
        refused(yuuka_gemm_quant(&stream, at(0, 0), 0, at(1, 0), 0, YUUKA_DTYPE_F32, at(2, 1), 0, type, 256, 4, 1, YUUKA_GEMM_PATH_AUTO, 0, nullptr), "the weights",
                "gemm_quant, GGUF order", 1);
    refused(yuuka_gemm_quant(&stream, at(0, 0), 0, at(1, 0), 0, YUUKA_DTYPE_F32, at(2, 2), 0, YUUKA_DTYPE_F32, 256, 4, 1, YUUKA_GEMM_PATH_AUTO, 0, nullptr),
            "the weights", "gemm_quant, f32", 2);
    for (int s : {1, 2, 3}) {
        const int32_t tokens[2] = {1, 2};
        const float uniforms[4] = {0.5f, 0.5f, 0.5f, 0.5f};
        int32_t accepted[1], emitted[2];
        refused(yuuka_accept_tree(&stream, at(0, s), 1, 2, 100, tokens, nullptr, YUUKA_ACCEPT_GREEDY, 0.0f, nullptr, nullptr, accepted, emitted, nullptr, nullptr, nullptr),
                "logits", "accept_tree", s);
        refused(yuuka_accept_tree(&stream, at(0, 0), 1, 2, 100, tokens, nullptr, YUUKA_ACCEPT_REJECTION, 1.0f, at(1, s), uniforms, accepted, emitted, nullptr, nullptr,
                                  nullptr),
                "draft_probs", "accept_tree", s);
        refused(yuuka_spec_lookup_draft_device(&stream, at(0, s), 10, 4, 2, at(1, 0)), "history", "lookup_draft_device", s);
        refused(yuuka_spec_lookup_draft_device(&stream, at(0, 0), 10, 4, 2, at(1, s)), "out", "lookup_draft_device", s);
    }
    printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures != 0;
}
