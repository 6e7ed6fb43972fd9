// Attention over the 4-bit key/value cache: argument checks, choice of kernel, workspace.
#include "internal.h"
#include "kv4.cuh"
#include "kv4_decode.cuh"
#include "kv4_chunk.cuh"
#include "../../include/decdec_b200.h"

#include <cmath>
#include <cstdio>

namespace dd {
namespace {

int fail(int code, const char* fmt, unsigned long long a = 0, unsigned long long b = 0) {
    char msg[256];
    snprintf(msg, sizeof(msg), fmt, a, b);
    return set_last_error(code, msg);
}

// Which kernel, and how many blocks fill the device.
struct Choice {
    bool chunk;                 // tiles of 256 rows on the fifth-generation tensor cores
    uint32_t nt;                // else tiles of 8 nt rows
    uint32_t blocks;
    size_t bytes;               // of the workspace
};

// Tiles of 8 rows while a request's rows (queries x heads of a key head) fit one, of 16 up to 64 rows, then of 256; heads of 256 elements
// have no registers for 16 and no room for 256.  Measured (us; 16 requests of 4096 tokens, 8 key heads of 128) with tiles of 16 / of 256: 32
// rows 63 / 105, 64 rows 108 / 114, 96 rows 150 / 124; with a step for 32 elements 90 / 108, 160 / 117, 226 / 126; one request of
// 32768 tokens 39 / 64, 59 / 68, 78 / 73.  One choice for the batch, by its largest request: the host does not know the others.
int choose(uint32_t head_dim, uint32_t group, uint32_t ratio, uint32_t max_queries, int dt, Choice* c) {
    const uint64_t rows = (uint64_t)ratio * max_queries;
    c->chunk = head_dim <= 128 && ratio <= (uint32_t)kChunkRows && rows > 64;
    c->nt = c->chunk ? kChunkRows / 8 : head_dim <= 128 && rows > 8 ? 2 : 1;
    c->blocks = device_sms();
    if (!c->chunk) {
        const int per_sm = head_dim == 64 ? kv4_decode64_blocks_per_sm(group, c->nt, dt) : head_dim == 128 ? kv4_decode128_blocks_per_sm(group, c->nt, dt)
                                                                                                           : kv4_decode256_blocks_per_sm(group, c->nt, dt);
        if (per_sm < 1) return fail(DECDEC_E_CUDA, "the attention kernel does not fit the current device");
        c->blocks *= (uint32_t)per_sm;
    }
    c->bytes = (size_t)c->blocks * (2u * kv4_part_floats(head_dim, c->nt) * sizeof(float) + sizeof(Kv4Cut));
    return 0;
}

int check(uint32_t requests, uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t group, uint32_t max_queries, int dtype) {
    if (dtype != FP16 && dtype != BF16) return fail(DECDEC_E_INVALID, "the 4-bit cache supports half and bfloat16 only.");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(DECDEC_E_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %llu", head_dim);
    if ((group != 32 && group != 64 && group != 128) || group > head_dim)
        return fail(DECDEC_E_INVALID, "group_size must be 32, 64 or 128 and not above head_dim, got %llu", group);
    if (kv_heads == 0 || heads == 0 || heads % kv_heads) return fail(DECDEC_E_INVALID, "heads must be a multiple of kv_heads (%llu, %llu)", heads, kv_heads);
    if (max_queries == 0) return fail(DECDEC_E_INVALID, "max_queries must be at least 1");
    if (requests > 0x7ffffffeu || (uint64_t)rows * heads > 0x7fffffffull) return fail(DECDEC_E_UNSUPPORTED, "too many requests or rows");
    return 0;
}

}  // namespace
}  // namespace dd

using namespace dd;

extern "C" {

int decdec_kv4_attention_workspace(uint32_t requests, uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                                   uint32_t max_queries, int dtype, size_t* bytes) {
    if (!bytes) return fail(DECDEC_E_INVALID, "null output pointer");
    if (int r = check(requests, rows, heads, kv_heads, head_dim, group_size, max_queries, dtype)) return r;
    Choice c;
    if (int r = choose(head_dim, group_size, heads / kv_heads, max_queries, dtype, &c)) return r;
    *bytes = c.bytes;
    return 0;
}

int decdec_kv4_attention(const void* q, int64_t q_token, int64_t q_head, void* out, int64_t out_token, int64_t out_head, float* lse, const void* cache,
                         uint32_t pages, uint32_t page_size, const int32_t* table, int64_t table_stride, uint32_t table_cols, const int32_t* lengths,
                         const int32_t* query_starts, uint32_t requests, uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                         uint32_t group_size, uint32_t max_queries, float scale, uint32_t window, int clear_rest, void* workspace,
                         size_t workspace_bytes, int dtype, void* stream) {
    if (int r = check(requests, rows, heads, kv_heads, head_dim, group_size, max_queries, dtype)) return r;
    if (page_size == 0 || page_size % kCellTokens || page_size > 65536u)
        return fail(DECDEC_E_INVALID, "page_size must be a multiple of 16 up to 65536, got %llu", page_size);
    if (pages == 0 || pages > 0x7fffffffu) return fail(DECDEC_E_INVALID, "empty cache or too many pages");
    if ((uint64_t)pages * kv_heads * (page_size / kCellTokens) >= kNoCell) return fail(DECDEC_E_UNSUPPORTED, "the cache has more cells than 32 bits count");
    if ((uint64_t)table_cols * page_size > 0x7ffffe00ull) return fail(DECDEC_E_INVALID, "the tokens of a table row must stay below 2^31 - 512");
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(DECDEC_E_INVALID, "scale must be a positive number");
    if (rows == 0) return 0;
    if (!q || !out || !cache || (requests && (!lengths || !query_starts)) || (requests && table_cols && !table)) return fail(DECDEC_E_INVALID, "null pointer argument");
    if (reinterpret_cast<uintptr_t>(cache) & 15u) return fail(DECDEC_E_INVALID, "the cache must be 16-byte aligned device memory");
    if ((reinterpret_cast<uintptr_t>(out) & 7u) || out_token % 4 || out_head % 4) return fail(DECDEC_E_INVALID, "output rows must be 8-byte aligned");
    const uint32_t ratio = heads / kv_heads;
    Choice c;
    if (int r = choose(head_dim, group_size, ratio, max_queries, dtype, &c)) return r;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < c.bytes)
        return fail(DECDEC_E_INVALID, "workspace must be 16-byte aligned and hold what decdec_kv4_attention_workspace says");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    Kv4Attn p = {};
    if (int r = stream_error_word(s, &p.err)) return r;
    p.q = Rows{q, q_token, q_head};
    p.out = out; p.out_token = out_token; p.out_head = out_head;
    p.lse = lse;
    p.cache = reinterpret_cast<const uint8_t*>(cache);
    p.table = table; p.table_stride = table_stride; p.table_cols = table_cols;
    p.lengths = lengths; p.starts = query_starts;
    p.part = reinterpret_cast<float*>(workspace);
    p.pages = pages; p.page_cells = page_size / kCellTokens; p.page_bytes = p.page_cells * kv4_cell_bytes(head_dim, group_size);
    p.requests = requests; p.rows = rows; p.kv_heads = kv_heads; p.ratio = ratio;
    p.window = window > 0x7fffffffu ? 0u : window;
    p.q_vec = (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && q_token % 8 == 0 && q_head % 8 == 0;
    p.clear_rest = clear_rest ? 1u : 0u;
    p.scale_log2 = scale * 1.4426950408889634f;
    cudaError_t e;
    if (c.chunk) {
        e = launch_kv4_chunk(head_dim, group_size, dtype, p, c.blocks, s);
    } else {
        // no more blocks than the longest contexts that the table holds could give two cells a warp
        const uint64_t tiles = ((uint64_t)rows * ratio + 8u * c.nt - 1) / (8u * c.nt) + requests;
        const uint64_t cells = tiles * kv_heads * ((uint64_t)table_cols * p.page_cells + 1u);
        uint64_t blocks = (cells + 2 * kDecodeWarps - 1) / (2 * kDecodeWarps);
        if (blocks < tiles * kv_heads) blocks = tiles * kv_heads;               // a block for every segment
        if (blocks > c.blocks) blocks = c.blocks;
        if (blocks == 0) blocks = 1;
        e = head_dim == 64    ? launch_kv4_decode64(group_size, c.nt, dtype, p, (uint32_t)blocks, s)
            : head_dim == 128 ? launch_kv4_decode128(group_size, c.nt, dtype, p, (uint32_t)blocks, s)
                              : launch_kv4_decode256(group_size, c.nt, dtype, p, (uint32_t)blocks, s);
    }
    if (e != cudaSuccess) {
        char msg[256];
        snprintf(msg, sizeof(msg), "attention launch failed: %s", cudaGetErrorString(e));
        return set_last_error(DECDEC_E_CUDA, msg);
    }
    return 0;
}

}  // extern "C"
