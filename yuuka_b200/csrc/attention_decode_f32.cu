// Attention of one new token per sequence over pools in F32.
#include "attention_decode.cuh"

namespace yk {

void launch_decode_f32(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int sms) {
    (void)cols;  // eight: the sums, queries and two parts of everything fill the registers
    launch_decode_dims<YUUKA_KV_F32, 1>(s, p, head_dim, sms);
}

}  // namespace yk
