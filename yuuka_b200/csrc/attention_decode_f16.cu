// Attention of one new token per sequence over pools in F16.
#include "attention_decode.cuh"

namespace yk {

void launch_decode_f16(cudaStream_t s, const DecodeParams & p, int head_dim, int cols, int sms) {
    if (cols == 8) launch_decode_dims<YUUKA_KV_F16, 1>(s, p, head_dim, sms);
    else launch_decode_dims<YUUKA_KV_F16, 2>(s, p, head_dim, sms);
}

}  // namespace yk
