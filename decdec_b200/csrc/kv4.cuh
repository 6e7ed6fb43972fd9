// The 4-bit key/value cache: its format, and the launch interface of the kernels that write and read it.
//
// The cache is [pages][kv_heads][bytes of a page]; a page is a run of cells of 16 tokens.  A cell of a head of D elements with
// G elements per step holds
//   key codes    8 D bytes   [D/128][16 tokens][4][words of 32][2] 16-bit words of four codes: element = 128 b + 32 w + 8 [4] + 4 [2] + code
//   value codes  8 D bytes   [D/128][token / 8][8][token % 8 / 2][words of 64][2][token % 2]: element = 128 b + 64 w + 32 [2] + 4 [8] + code
//   key steps    64 D/G bytes [16 tokens][D/G] pairs (step, offset) of the 16-bit type
//   value steps  64 D/G bytes the same
// and an element is offset + step * code.  The order is that of the tensor-core operands that attention makes of it (mma.m16n8k16):
// a lane finds its keys' codes (rows = tokens, pairs along the head) and its values' codes (rows = elements, pairs along the tokens)
// in 16 consecutive bytes each, and a mask over a word leaves two codes in the halves that become a pair of factors (kv4_decode.cuh).
#pragma once
#include "common.cuh"

#include <cstdlib>
#include <utility>

namespace dd {

constexpr int kCellTokens = 16;
// codes in the error word of a stream, beside those of the GEMVs
constexpr unsigned kErrKv4Page = 3;       // a page or a slot outside the cache, or a length beyond the block table

__host__ __device__ constexpr uint32_t kv4_cell_bytes(uint32_t d, uint32_t group) { return 16u * (d + 8u * (d / group)); }

// byte of the 16-bit word that holds elements 4u .. 4u+3 of token r (0..15) of a cell
__host__ __device__ constexpr uint32_t kv4_key_word(uint32_t d, uint32_t r, uint32_t u) {
    const uint32_t per = d < 128u ? d / 32u : 4u;             // words of 32 elements in a block
    const uint32_t b = u / 32u, w = u / 8u % per, four = u % 8u / 2u, half = u % 2u;
    return (((b * 16u + r) * 4u + four) * per + w) * 4u + half * 2u;
}
__host__ __device__ constexpr uint32_t kv4_value_word(uint32_t d, uint32_t r, uint32_t u) {
    const uint32_t per = d < 128u ? d / 64u : 2u;             // words of 64 elements in a block
    const uint32_t b = u / 32u, w = u / 16u % per, half = u / 8u % 2u, eight = u % 8u;
    return 8u * d + ((((b * 2u + r / 8u) * 8u + eight) * 4u + r % 8u / 2u) * per + w) * 8u + half * 4u + (r % 2u) * 2u;
}
__host__ __device__ constexpr uint32_t kv4_key_step(uint32_t d, uint32_t group, uint32_t r, uint32_t g) {
    return 16u * d + (r * (d / group) + g) * 4u;
}
__host__ __device__ constexpr uint32_t kv4_value_step(uint32_t d, uint32_t group, uint32_t r, uint32_t g) {
    return 16u * d + 64u * (d / group) + (r * (d / group) + g) * 4u;
}

template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typename Tr<DT>::T v[2] = {Tr<DT>::from_f(a), Tr<DT>::from_f(b)};
    return *reinterpret_cast<const uint32_t*>(v);
}

// rows [tokens][heads][head_dim] of a 16-bit type, strides in elements
struct Rows {
    const void* p;
    long long token, head;
};

struct Kv4Cache {
    uint8_t* data;
    uint32_t pages, page_cells, kv_heads, head_dim, group;
    uint32_t page_bytes;                  // of one head
};

struct Kv4Attn {
    Rows q;
    void* out;
    long long out_token, out_head;
    float* lse;                           // [rows][heads] or null
    const uint8_t* cache;
    const int32_t* table;
    long long table_stride;
    const int32_t* lengths;
    const int32_t* starts;
    float* part;                          // sums of cut segments: see kv4_decode.cuh
    unsigned* err;
    uint32_t pages, page_cells, page_bytes, table_cols;
    uint32_t requests, rows, kv_heads, ratio;
    uint32_t window;
    uint32_t q_vec;                       // queries may be read 16 bytes at a time
    uint32_t clear_rest;                  // rows of no request are cleared
    float scale_log2;                     // scale of the scores * log2(e)
};

cudaError_t launch_rotary(int dt, const Rows& q, uint32_t q_heads, const Rows& k, uint32_t k_heads, void* q_out, long long qo_token,
                          long long qo_head, void* k_out, long long ko_token, long long ko_head, const void* positions, int wide,
                          const double* frequencies, uint32_t tokens, uint32_t head_dim, uint32_t rotary_dim, int interleaved,
                          float factor, cudaStream_t s);

// Decode attention, 8 nt query rows (queries x heads of a key head) in a tile: blocks that fit an SM (0: no such kernel), and the launch
#define KV4_DECODE(D_)                                                                    \
    int kv4_decode##D_##_blocks_per_sm(uint32_t group, uint32_t nt, int dt);              \
    cudaError_t launch_kv4_decode##D_(uint32_t group, uint32_t nt, int dt, const Kv4Attn& p, uint32_t blocks, cudaStream_t s)
KV4_DECODE(64);
KV4_DECODE(128);
KV4_DECODE(256);
#undef KV4_DECODE

// Attention of many queries, heads of 64 and 128: one block an SM
cudaError_t launch_kv4_chunk(uint32_t head_dim, uint32_t group, int dt, const Kv4Attn& p, uint32_t blocks, cudaStream_t s);

// A launch whose blocks may become resident while the previous kernel of the stream drains (every kernel here waits for it before
// it reads anything); DECDEC_PDL=0 turns that off.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args&&... args) {
    static const bool early = [] {
        const char* v = getenv("DECDEC_PDL");
        return !(v && v[0] == '0');
    }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

int stream_error_word(cudaStream_t s, unsigned** err);    // 0, or the code that the call has to return

}  // namespace dd
