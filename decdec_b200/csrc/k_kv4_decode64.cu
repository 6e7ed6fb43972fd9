// Decode attention over the 4-bit cache, heads of 64 elements.
#include "kv4_decode.cuh"

namespace dd {

int kv4_decode64_blocks_per_sm(uint32_t group, uint32_t nt, int dt) { return for_decode<64>(group, nt, dt, BlocksCall<64>{}); }

cudaError_t launch_kv4_decode64(uint32_t group, uint32_t nt, int dt, const Kv4Attn& p, uint32_t blocks, cudaStream_t s) {
    return for_decode<64>(group, nt, dt, DecodeCall<64>{p, blocks, s});
}

}  // namespace dd
