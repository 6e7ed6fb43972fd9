// Decode attention over the 4-bit cache, heads of 256 elements.
#include "kv4_decode.cuh"

namespace dd {

int kv4_decode256_blocks_per_sm(uint32_t group, uint32_t nt, int dt) { return for_decode<256>(group, nt, dt, BlocksCall<256>{}); }

cudaError_t launch_kv4_decode256(uint32_t group, uint32_t nt, int dt, const Kv4Attn& p, uint32_t blocks, cudaStream_t s) {
    return for_decode<256>(group, nt, dt, DecodeCall<256>{p, blocks, s});
}

}  // namespace dd
