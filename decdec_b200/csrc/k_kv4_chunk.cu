// Attention of many queries over the 4-bit cache.
#include "kv4_chunk.cuh"

namespace dd {

cudaError_t launch_kv4_chunk(uint32_t head_dim, uint32_t group, int dt, const Kv4Attn& p, uint32_t blocks, cudaStream_t s) {
#define KV4_CASE(D_, G_) \
    if (head_dim == D_ && group == G_) return dt == FP16 ? run_chunk<D_, G_, FP16>(p, blocks, s) : run_chunk<D_, G_, BF16>(p, blocks, s)
    KV4_CASE(64, 32);
    KV4_CASE(64, 64);
    KV4_CASE(128, 32);
    KV4_CASE(128, 64);
    KV4_CASE(128, 128);
#undef KV4_CASE
    return cudaErrorInvalidValue;
}

}  // namespace dd
