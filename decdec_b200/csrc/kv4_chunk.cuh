// Attention of many queries over the 4-bit cache (prompts in chunks, long drafts): tiles of 256 query rows on the fifth-generation
// tensor cores.
//
// Per tile and step of 128 tokens, S = Q K^T and O += P V with fp16 operands and fp32 sums in tensor memory.  Keys and values become
// fp16 numbers on the way (offset + step * code in one rounding, 2^-11, as a gathered cache in 16 bits has; scaled by a power of two per
// 32 tokens so that both 16-bit types fit), once for the 256 rows of a tile.  Bound by the products and the exponentials: for heads of 128, a step
// of a tile is 2048 cycles of each; it takes 6100, most of it the chain maximum -> exponentials -> products of a group.  17 warps leave a thread 96
// registers, and every instance spills (152 to 216 bytes of stores).  Three requests with chunks of up to 2048 queries at up to 16384 tokens:
// 1.24 ms, 697 TFLOP/s.
//
// A weight carries the power of two by which its 32 tokens' values are smaller than the largest of the request's steps so far: where that passes 2^14 the
// fp16 weights are subnormal, and outputs are good to 2^-28 of those largest values a token, whether the row sees them or not.  Sums of
// weights are fp32 and keep theirs.
//
// One block an SM, 17 warps:
//   warps 0-3, 4-7   rows 0-127 and 128-255 of the tile, a thread a row: queries into shared memory; per step the row's maximum and sum,
//                    P = exp2(S - maximum) written over S as fp16; sums rescaled when a maximum has grown by 2^8; output at the end.  One group
//                    computes while the products of the other run.
//   warps 8-11       key codes from the cache (registers, a step ahead) to fp16 tiles in shared memory, two stages; a warp 32 tokens
//   warps 12-15      value codes the same
//   warp 16          issues the products
// The work is a line of (request, tile, head, 128 tokens) cut evenly over the blocks as in kv4_decode.cuh; parts of cut segments are joined
// by the same kernel.
//
// Shared memory: operands as rows of 128 bytes, eight rows to a 1024-byte atom, 16-byte chunks exchanged by row (the 128-byte swizzle).
// Elements of a head lie in the order in which a word of key codes unpacks (within eight: 0 4 1 5 2 6 3 7), in queries and keys alike; rows of
// the transposed values so that eight neighbouring lanes write eight neighbouring rows (32 i + 8 j + [8] for element 32 i + 4 [8] + j).
//
// Waits are bounded: one that runs out raises error 1 of the stream and turns all others off, and the block runs through to its end.
#pragma once
#include "kv4_decode.cuh"

namespace dd {

constexpr int kChunkRows = 256, kChunkStep = 128, kChunkThreads = 17 * 32;
constexpr float kChunkGrow = 8.0f;
constexpr int kSegmentSteps = 2;              // what a segment's beginning and end count on the line, in steps (counted as none: 2 % slower; heads of 128)
constexpr unsigned kErrWait = 1;
constexpr long long kWaitClocks = 1000000000;    // about half a second

struct ChunkRequest {
    int start, queries, length, tiles, per_tile;         // per_tile: queries of a tile
};
struct ChunkTile {
    int q0, n;                                            // queries of the tile
    int from, steps;                                      // first step of 128 tokens that some row sees, number (at least one)
};

__device__ __forceinline__ ChunkRequest chunk_request(const Kv4Attn& p, uint32_t b, bool report) {
    ChunkRequest r;
    const int rows = (int)p.rows;
    r.start = min(max(p.starts[b], 0), rows);
    r.queries = max(min(max(p.starts[b + 1], 0), rows) - r.start, 0);
    r.length = max(p.lengths[b], 0);
    const long long most = (long long)p.table_cols * p.page_cells * kCellTokens;
    if ((long long)r.length > most) {
        if (report) raise_error(p.err, kErrKv4Page);
        r.length = (int)most;
    }
    r.per_tile = kChunkRows / (int)p.ratio;
    r.tiles = (r.queries + r.per_tile - 1) / r.per_tile;
    return r;
}
__device__ __forceinline__ ChunkTile chunk_tile(const Kv4Attn& p, const ChunkRequest& r, int t) {
    ChunkTile c;
    c.q0 = t * r.per_tile;
    c.n = min(r.per_tile, r.queries - c.q0);
    const long long pos = (long long)r.length - r.queries + c.q0;                       // of the first query
    const int end = (int)max(0ll, pos + c.n);                                           // tokens below it are seen
    c.from = p.window ? (int)(max(0ll, pos - (long long)p.window + 1) / kChunkStep) : 0;
    c.steps = max(1, (end + kChunkStep - 1) / kChunkStep - c.from);
    return c;
}

// ---- fifth-generation tensor cores: operands in shared memory (64-bit descriptors) or tensor memory, sums in tensor memory
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// rows of 128 bytes, eight rows 1024 bytes, 128-byte swizzle
__device__ __forceinline__ uint64_t operand(uint32_t at) {
    return (uint64_t)((at >> 4) & 0x3fffu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// fp16 x fp16 -> fp32, both operands with the depth contiguous, 128 rows, n columns
__host__ __device__ constexpr uint32_t product_shape(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(add) : "memory");
}
__device__ __forceinline__ void product_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"(add) : "memory");
}
__device__ __forceinline__ void products_done(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
                   "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// what this thread wrote to shared memory is seen by products issued after a barrier that it arrives on next
__device__ __forceinline__ void operands_written() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded: then the block gives up, here and in every later wait.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* gave_up, unsigned* err) {
    if (bar_try(bar, parity)) return;
    const long long t0 = clock64();
    while (!bar_try(bar, parity)) {
        if (*gave_up) return;
        if (clock64() - t0 > kWaitClocks) {
            *gave_up = 1u;
            raise_error(err, kErrWait);
            return;
        }
    }
}

template <int D> struct ChunkShape {
    static constexpr uint32_t kBlocks = D / 64;                                  // 128-byte rows to a row of D elements
    static constexpr uint32_t kQ = kChunkRows * D * 2, kK = kChunkStep * D * 2, kV = kChunkStep * D * 2;
    static constexpr uint32_t kBytes = kQ + 2 * kK + 2 * kV + 1024u;             // and the way to a 1024-byte boundary
};

// per step of 128 tokens, from the converting warps to the rows, by 32 tokens: exponents of keys and values, tokens whose values are no
// numbers in any group and by group
struct __align__(16) ChunkMeta {
    int key_exp[4], value_exp[4];
    uint32_t any_poison[4], poison[4][4];
};

template <int D, int GS, int DT>
__global__ void __launch_bounds__(kChunkThreads, 1) kv4_chunk_kernel(Kv4Attn p) {
    using T = typename Tr<DT>::T;
    using Sh = ChunkShape<D>;
    constexpr int NG = D / GS;
    constexpr uint32_t CELL = kv4_cell_bytes(D, GS);
    constexpr int LW = D / 32;                                                   // 16-byte loads of a lane's keys (and values) in a step
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[15];
    __shared__ uint32_t s_tmem, s_gave_up;
    __shared__ ChunkMeta s_meta[4];
    __shared__ long long s_sum[17];
    __shared__ int s_seg[4];                                                     // request, tile, head, step within the segment

    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t bar0 = smem_at(bars);
    const uint32_t bar_k = bar0, bar_kfree = bar0 + 16, bar_v = bar0 + 32, bar_vfree = bar0 + 48, bar_s = bar0 + 64, bar_p = bar0 + 80, bar_o = bar0 + 96;
    const uint32_t bar_q = bar0 + 104, bar_end = bar0 + 112;                     // one for the outputs of both groups, the queries, the end
    volatile uint32_t* gave_up = &s_gave_up;

    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_at(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        s_gave_up = 0u;
        for (int i = 0; i < 2; ++i) {
            bar_init(bar_k + 8 * i, 4);
            bar_init(bar_kfree + 8 * i, 1);
            bar_init(bar_v + 8 * i, 4);
            bar_init(bar_vfree + 8 * i, 1);
            bar_init(bar_s + 8 * i, 2);
            bar_init(bar_p + 8 * i, 4);
        }
        bar_init(bar_o, 1);                                                      // both groups' outputs end together
        bar_init(bar_q, 8);
        bar_init(bar_end, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_trigger();
    pdl_wait();

    // ---- this block's part of the line: a warp sums a run of requests, its lanes their tiles
    const uint32_t run = (p.requests + 16u) / 17u;
    const uint32_t rb0 = min(warp * run, p.requests), rb1 = min(rb0 + run, p.requests);
    auto total_of = [&](const ChunkRequest& r) {
        long long n = 0;
        for (int t = lane; t < r.tiles; t += 32) n += chunk_tile(p, r, t).steps + kSegmentSteps;
#pragma unroll
        for (int o = 16; o; o /= 2) n += __shfl_xor_sync(0xffffffffu, n, o);
        return n * p.kv_heads;
    };
    long long mine = 0;
    for (uint32_t b = rb0; b < rb1; ++b) mine += total_of(chunk_request(p, b, blockIdx.x == 0 && lane == 0));
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    long long before = 0, total = 0;
    for (int w = 0; w < 17; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    // at least two steps a block: a shorter part would spend its time in the joining of the parts
    const long long per = max((long long)ratio_of(total + gridDim.x - 1, gridDim.x), 2ll);
    const long long x0 = (long long)blockIdx.x * per, x1 = min(x0 + per, total);
    if (x0 < x1 && before <= x0 && x0 < before + mine) {
        long long at = before;
        uint32_t b = rb0;
        ChunkRequest r;
        for (;; ++b) {                                                           // ends: x0 lies below the end of this run
            r = chunk_request(p, b, false);
            const long long n = total_of(r);
            if (x0 < at + n) break;
            at += n;
        }
        for (int t0 = 0;; t0 += 32) {                                            // ends: x0 lies below the end of the request
            const int t = t0 + lane, steps = t < r.tiles ? chunk_tile(p, r, t).steps + kSegmentSteps : 0;
            const long long n = (long long)steps * p.kv_heads;
            long long incl = n;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const long long v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const bool here = x0 >= at + incl - n && x0 < at + incl;
            if (here) {
                const long long in = x0 - (at + incl - n);
                s_seg[0] = (int)b; s_seg[1] = t;
                s_seg[2] = (int)ratio_of(in, steps);
                s_seg[3] = (int)(in - (long long)s_seg[2] * steps);
            }
            if (__any_sync(0xffffffffu, here)) break;
            at += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s_tmem;
    if (p.clear_rest) clear_rest<D, DT>(p, tid, kChunkThreads);

    // ---- the segments, walked by every warp for itself
    struct Segment {
        uint32_t b;
        ChunkRequest r;
        ChunkTile t;
        int tile, head, c0, c1, pos, take;                                       // pos, take: of its part of the line
        long long x;
    } g;
    auto range = [&] {
        g.take = (int)min((long long)(g.t.steps + kSegmentSteps - g.pos), x1 - g.x);
        g.c0 = max(g.pos - kSegmentSteps, 0);
        g.c1 = max(g.pos + g.take - kSegmentSteps, 0);
    };
    auto first = [&] {
        g.x = x0;
        if (x0 >= x1) return;
        g.b = (uint32_t)s_seg[0]; g.tile = s_seg[1]; g.head = s_seg[2]; g.pos = s_seg[3];
        g.r = chunk_request(p, g.b, false);
        g.t = chunk_tile(p, g.r, g.tile);
        range();
    };
    auto next = [&] {
        g.x += g.take;
        if (g.x >= x1) return;
        g.pos = 0;
        if (++g.head == (int)p.kv_heads) {
            g.head = 0;
            if (++g.tile == g.r.tiles) {
                g.tile = 0;
                do g.r = chunk_request(p, ++g.b, false); while (g.r.tiles == 0);      // ends: work remains
            }
            g.t = chunk_tile(p, g.r, g.tile);
        }
        range();
    };
    // a range that ends before the first step of its last segment leaves that to the next block
    auto more = [&] { return g.x < x1 && g.c1 > g.c0; };
    const uint32_t smem_s = smem_at(smem), smem_k = smem_s + Sh::kQ, smem_v = smem_k + 2 * Sh::kK;

    if (warp == 16) {
        // ================================ products ================================
        if (lane == 0) {
            uint32_t step = 0, seg = 0, turn[2] = {0, 0};                        // steps of this block; steps of each group
            const uint32_t shape_s = product_shape(kChunkStep), shape_o = product_shape(D);
            const uint64_t at_q = operand(smem_s), at_k = operand(smem_k), at_v = operand(smem_v);       // addresses count 16 bytes
            auto scores = [&](uint32_t grp, uint32_t stage) {
                const uint64_t a = at_q + grp * (128u * 128u / 16u), b = at_k + stage * (Sh::kK / 16u);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    product(tmem + 2 * D + grp * 128u, a + (k / 4) * (kChunkRows * 8u) + (k % 4) * 2u, b + (k / 4) * (kChunkStep * 8u) + (k % 4) * 2u, shape_s, k > 0);
                products_done(bar_s + 8 * grp);
                bar_arrive(bar_s + 8 * grp);                                     // what the key warps left for the rows is visible with it
            };
            for (first(); more(); next()) {
                const uint32_t groups = g.t.n * (int)p.ratio > 128 ? 2u : 1u;
                const int steps = g.c1 - g.c0;
                bar_wait(bar_q, seg & 1u, gave_up, p.err);
                bar_wait(bar_k + 8 * (step & 1u), (step >> 1) & 1u, gave_up, p.err);
                tc_after();
                for (uint32_t i = 0; i < groups; ++i) scores(i, step & 1u);
                products_done(bar_kfree + 8 * (step & 1u));
                for (int j = 0; j < steps; ++j, ++step) {
                    const uint32_t stage = step & 1u, ahead = (step + 1u) & 1u;
                    for (uint32_t i = 0; i < groups; ++i) {
                        bar_wait(bar_p + 8 * i, turn[i] & 1u, gave_up, p.err);
                        ++turn[i];
                        if (i == 0) bar_wait(bar_v + 8 * stage, (step >> 1) & 1u, gave_up, p.err);
                        tc_after();
#pragma unroll
                        for (int k = 0; k < kChunkStep / 16; ++k)
                            product_from_tmem(tmem + i * D, tmem + 2 * D + i * 128u + k * 8u,
                                              at_v + stage * (Sh::kV / 16u) + (k / 4) * (D * 8u) + (k % 4) * 2u, shape_o, j > 0 || k > 0);
                        if (j + 1 < steps) {
                            if (i == 0) {
                                bar_wait(bar_k + 8 * ahead, ((step + 1u) >> 1) & 1u, gave_up, p.err);
                                tc_after();
                            }
                            scores(i, ahead);                                    // over P, which the products before it have read
                        }
                    }
                    products_done(bar_vfree + 8 * stage);
                    if (j + 1 < steps) products_done(bar_kfree + 8 * ahead);
                }
                products_done(bar_o);
                ++seg;
            }
            // A block that gave up issued products that nobody waits for: they end before the tensor memory is freed and the block leaves.
            products_done(bar_end);
            const long long t0 = clock64();
            while (!bar_try(bar_end, 0u) && clock64() - t0 < kWaitClocks) {}
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ================================ codes to numbers ================================
        const bool values = warp >= 12;
        const int w4 = warp & 3, t = w4 * 32 + lane;                             // token of the step; also (cell, half of its tokens, eight) of the values
        uint32_t step = 0;
        struct Raw {
            uint4 x[LW];                                                         // the keys' row; the values of eight tokens at every eighth element
            uint32_t s[NG];                                                      // the token's steps
        };
        // page of the thread's cell of a step; -1 behind the end
        auto page_of = [&](int block) {
            const int tok = block * kChunkStep + (t & ~15);
            return tok < g.r.length ? p.table[(long long)g.b * p.table_stride + (uint32_t)tok / kCellTokens / p.page_cells] : -1;
        };
        // Coherent loads past the first-level cache: this block may have become resident before an append that it waited for wrote these bytes,
        // which loads of read-only memory do not allow.
        auto load = [&](Raw& x, int page, int block) {
            const uint32_t r = t & 15, c = (uint32_t)(block * kChunkStep + t) / kCellTokens;
#pragma unroll
            for (int i = 0; i < LW; ++i) x.x[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < NG; ++i) x.s[i] = 0u;
            if (page < 0 || (uint32_t)page >= p.pages) {
                if (block * kChunkStep + (t & ~15) < g.r.length) raise_error(p.err, kErrKv4Page);
                return;
            }
            const uint8_t* cell = p.cache + ((size_t)page * p.kv_heads + g.head) * p.page_bytes + (size_t)(c % p.page_cells) * CELL;
#pragma unroll
            for (int i = 0; i < LW; ++i) x.x[i] = __ldcg(reinterpret_cast<const uint4*>(cell + (values ? 8 * D : 0) + r * (D / 2)) + i);
            if (block * kChunkStep + t < g.r.length) {                           // else what the page held before
#pragma unroll
                for (int i = 0; i < NG; ++i)
                    x.s[i] = __ldcg(reinterpret_cast<const uint32_t*>(cell + (values ? kv4_value_step(D, GS, r, i) : kv4_key_step(D, GS, r, i))));
            }
        };
        auto word = [](const Raw& x, int at) {
            const uint4& q = x.x[at / 4];
            return at % 4 == 0 ? q.x : at % 4 == 1 ? q.y : at % 4 == 2 ? q.z : q.w;
        };
        const uint32_t bar_full = values ? bar_v : bar_k, bar_free = values ? bar_vfree : bar_kfree;
        for (first(); more(); next()) {
            const int block0 = g.t.from + g.c0, steps = g.c1 - g.c0;
            Raw cur, ahead;
            int page = page_of(block0);
            int page1 = steps > 1 ? page_of(block0 + 1) : -1;
            load(cur, page, block0);
            int largest = -100;                                                  // exponent of the values so far
            for (int j = 0; j < steps; ++j, ++step) {
                const uint32_t stage = step & 1u;
                if (j + 1 < steps) {
                    load(ahead, page1, block0 + j + 1);
                    if (j + 2 < steps) page1 = page_of(block0 + j + 2);
                }
                // the largest magnitude of the warp's tokens that steps and offsets allow; what is no number does not count
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const float2 f = unpack2<DT>(cur.s[i]);
                    const float m = fmaxf(fabsf(f.y), fabsf(fmaf(15.0f, f.x, f.y)));        // a rounded step may lead beyond the largest number
                    if (fabsf(f.y) < INFINITY) top = fmaxf(top, fminf(m, 3.402823466e+38f));
                }
                int e = max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127, -100);
                ChunkMeta& meta = s_meta[step & 3u];
                if (!values) {
                    if (lane == 0) meta.key_exp[w4] = e;
                    const float by = pow2(12 - e);
                    if (step >= 2) bar_wait(bar_free + 8 * stage, ((step >> 1) - 1u) & 1u, gave_up, p.err);
                    uint8_t* row = smem + Sh::kQ + stage * Sh::kK + t * 128;
#pragma unroll
                    for (int w = 0; w < LW; ++w) {
                        const float2 st = unpack2<DT>(cur.s[w * 32 / GS]);
                        const __half2 a = __float2half2_rn(st.x * by), b = __float2half2_rn(fmaf(8.0f, st.x, st.y) * by);
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
                            uint32_t h[4];                                       // word (f, w): elements 32 w + 8 f .. + 7
                            code_pairs(word(cur, f * LW + w), h);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&h[i]), a, b);
                                h[i] = *reinterpret_cast<const uint32_t*>(&r);
                            }
                            const uint32_t chunk = w * 4 + f;
                            *reinterpret_cast<uint4*>(row + (chunk / 8) * (kChunkStep * 128) + ((chunk % 8) ^ (t & 7)) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    }
                } else {
                    largest = max(largest, e);
                    const float by = pow2(12 - largest);
                    uint32_t any = 0, mine[NG];                                  // (step, middle) of this token as fp16
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const float2 st = unpack2<DT>(cur.s[i]);
                        const bool number = fabsf(st.y) < INFINITY;              // values that are no numbers are left out and marked
                        mine[i] = number ? half2_bits(st.x * by, fmaf(8.0f, st.x, st.y) * by) : 0u;
                        const uint32_t poison = __ballot_sync(0xffffffffu, !number);
                        if (lane == 0) meta.poison[i][w4] = poison;
                        any |= poison;
                    }
                    if (lane == 0) { meta.any_poison[w4] = any; meta.value_exp[w4] = largest; }
                    if (step >= 2) bar_wait(bar_free + 8 * stage, ((step >> 1) - 1u) & 1u, gave_up, p.err);
                    uint8_t* base = smem + Sh::kQ + 2 * Sh::kK + stage * Sh::kV;
                    const int eight = t & 7, chunk = t >> 3;                     // 16-byte chunk of eight tokens: 16 of them to a row
#pragma unroll
                    for (int gr = 0; gr < NG; ++gr) {
                        uint32_t a[4], b[4];                                     // of the token pairs, which the eight lanes of the chunk own
#pragma unroll
                        for (int pr = 0; pr < 4; ++pr) {
                            const uint32_t u = __shfl_sync(0xffffffffu, mine[gr], (lane & 24) + 2 * pr), v = __shfl_sync(0xffffffffu, mine[gr], (lane & 24) + 2 * pr + 1);
                            a[pr] = __byte_perm(u, v, 0x5410);
                            b[pr] = __byte_perm(u, v, 0x7632);
                        }
#pragma unroll
                        for (int i = gr * GS / 32; i < (gr + 1) * GS / 32; ++i) {
                            uint32_t h[4][4];                                    // [pair of tokens][element j]
#pragma unroll
                            for (int pr = 0; pr < 4; ++pr) {
                                code_pairs(word(cur, pr * LW + i), h[pr]);       // words of a pair: LW of 32 elements
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&h[pr][x]), *reinterpret_cast<const __half2*>(&a[pr]),
                                                              *reinterpret_cast<const __half2*>(&b[pr]));
                                    h[pr][x] = *reinterpret_cast<const uint32_t*>(&r);
                                }
                            }
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const int row = 32 * i + 8 * x + eight;
                                *reinterpret_cast<uint4*>(base + (chunk / 8) * (D * 128) + row * 128 + ((chunk % 8) ^ eight) * 16) =
                                    make_uint4(h[0][x], h[1][x], h[2][x], h[3][x]);
                            }
                        }
                    }
                }
                operands_written();
                __syncwarp();
                if (lane == 0) bar_arrive(bar_full + 8 * stage);
                cur = ahead;
            }
        }
    } else {
        // ================================ rows ================================
        const uint32_t grp = warp >> 2;
        const int row = tid;                                                     // of the tile
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t at_s = tmem + 2 * D + grp * 128u + lanes, at_o = tmem + grp * D + lanes;
        uint32_t step = 0, seg = 0, turn = 0;
        Kv4Cut cut = {};
        for (first(); more(); next()) {
            const int live_rows = g.t.n * (int)p.ratio, steps = g.c1 - g.c0;
            const bool active = grp == 0 || live_rows > 128, live = row < live_rows;
            const int query = g.t.q0 + (live ? row / (int)p.ratio : 0), sub = live ? row % (int)p.ratio : 0;
            float sf;
            {
                // the row as fp16, scaled to a power of two near 2^13; read twice, to hold little of it
                const T* src = reinterpret_cast<const T*>(p.q.p) + (long long)(g.r.start + query) * p.q.token + ((long long)g.head * p.ratio + sub) * p.q.head;
                auto eight = [&](int c) {
                    if (!live) return make_uint4(0, 0, 0, 0);
                    if (p.q_vec) return *reinterpret_cast<const uint4*>(src + 8 * c);
                    const uint16_t* e = reinterpret_cast<const uint16_t*>(src + 8 * c);
                    return make_uint4((uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16, (uint32_t)e[4] | (uint32_t)e[5] << 16,
                                      (uint32_t)e[6] | (uint32_t)e[7] << 16);
                };
                float top = 0.0f;
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) {
                    const uint4 v = eight(c);
                    const float2 a = unpack2<DT>(v.x), b = unpack2<DT>(v.y), d = unpack2<DT>(v.z), f = unpack2<DT>(v.w);
                    top = fmaxf(fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y))),
                                fmaxf(fmaxf(fabsf(d.x), fabsf(d.y)), fmaxf(fabsf(f.x), fabsf(f.y))));
                }
                int e = (int)(__float_as_uint(top) >> 23) - 127;
                e = (top > 0.0f && top < INFINITY) ? max(e, -87) : 13;
                const float up = pow2(13 - e);
                sf = p.scale_log2 * pow2(e - 13);
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) {
                    const uint4 v = eight(c);
                    const float2 a = unpack2<DT>(v.x), b = unpack2<DT>(v.y), d = unpack2<DT>(v.z), f = unpack2<DT>(v.w);
                    *reinterpret_cast<uint4*>(smem + (c / 8) * (kChunkRows * 128) + row * 128 + ((c % 8) ^ (row & 7)) * 16) =
                        make_uint4(half2_bits(a.x * up, d.x * up), half2_bits(a.y * up, d.y * up), half2_bits(b.x * up, f.x * up), half2_bits(b.y * up, f.y * up));
                }
            }
            operands_written();
            __syncwarp();
            if (lane == 0) bar_arrive(bar_q);
            const long long pos = (long long)g.r.length - g.r.queries + query;
            const int to = live ? (int)max(pos + 1, 0ll) : 0, from = live && p.window ? (int)max(0ll, pos - (long long)p.window + 1) : 0;
            // steps between these are seen whole by every live row of the warp
            const int clear_to = __reduce_min_sync(0xffffffffu, live ? to : 0x7fffffff), clear_from = __reduce_max_sync(0xffffffffu, from);
            const bool any_live = __any_sync(0xffffffffu, live);
            float m = -INFINITY, l = 0.0f;
            int ev = 0;
            uint32_t bad = 0;                                                    // groups with a seen value that is no number
            for (int j = 0; j < steps; ++j, ++step) {
                if (!active) continue;
                bar_wait(bar_s + 8 * grp, turn & 1u, gave_up, p.err);
                ++turn;
                // The scores wait for the keys alone: the values' exponents and marks are there with the values of the step.  Their stage is not
                // filled again before this group has handed its weights over, so the phase cannot be missed.
                bar_wait(bar_v + 8 * (step & 1u), (step >> 1) & 1u, gave_up, p.err);
                tc_after();
                if (any_live) {
                    const ChunkMeta& meta = s_meta[step & 3u];
                    const int tok0 = (g.t.from + g.c0 + j) * kChunkStep;
                    const bool clear = tok0 >= clear_from && tok0 + kChunkStep <= clear_to;
                    const int4 ve = *reinterpret_cast<const int4*>(meta.value_exp);
                    int new_ev = max(max(ve.x, ve.y), max(ve.z, ve.w));
                    if (j > 0) new_ev = max(new_ev, ev);
                    // 32 tokens at a time, in a loop that is not unrolled: the roles' code has to stay in the instruction cache
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t r[32];
                        tmem_load32(at_s + 32 * c, r);
                        // above 0, or a hidden score of -inf times 0 would be NaN: keys of zeros (parts of a step without tokens) have the least exponent
                        const float f = fmaxf(sf * pow2(meta.key_exp[c] - 12), kLeastFactor);
                        // Weights times 2^(exponent of the values here - that of the sums).  Below -40 all of them (2^8 at most) are zeros in fp16 as
                        // well, and the sum, which is taken before that rounding, must not lose them: it keeps those above 2^-86.
                        const int shift = max(meta.value_exp[c] - new_ev, -40);
                        tmem_loaded();
                        if (!clear) {
                            const int lo = max(from - (tok0 + 32 * c), 0), hi = min(to - (tok0 + 32 * c), 32);
                            const uint32_t mask = lo >= hi ? 0u : (0xffffffffu >> (32 - (hi - lo))) << lo;
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((mask >> i) & 1u)) r[i] = 0xff800000u;             // -inf: a weight of 0
                        }
                        float top = __uint_as_float(r[0]);
#pragma unroll
                        for (int i = 1; i < 32; ++i) top = fmaxf(top, __uint_as_float(r[i]));
                        top *= f;
                        const bool follow = top > m + kChunkGrow || (c == 0 && j > 0 && new_ev != ev);
                        if (__any_sync(0xffffffffu, follow)) {
                            // rare after a segment's first steps: the sums, and the weights of the step that are written already, brought to
                            // another maximum or exponent.  Maxima are whole numbers, so that this is by powers of two: the fp16 weights of the step
                            // lose nothing by it but what becomes subnormal.
                            const float now = ceilf(fmaxf(m, top)), down = m == now ? 1.0f : m - now < -126.0f ? 0.0f : pow2((int)(m - now));
                            const float by = down * ex2((float)((j > 0 && c == 0 ? ev : new_ev) - new_ev));
                            m = now;
                            l *= down;
                            tmem_stored();
                            for (int k = 0; j > 0 && k < D / 8; ++k) {
                                uint32_t o[8];
                                tmem_load8(at_o + 8 * k, o);
                                tmem_loaded();
#pragma unroll
                                for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
                                tmem_store8(at_o + 8 * k, o);
                            }
                            const __half2 h = __float2half2_rn(down);
                            for (int k = 0; k < 2 * c; ++k) {
                                uint32_t o[8];
                                tmem_load8(at_s + 8 * k, o);
                                tmem_loaded();
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&o[i]), h);
                                    o[i] = *reinterpret_cast<const uint32_t*>(&x);
                                }
                                tmem_store8(at_s + 8 * k, o);
                            }
                        }
                        const float less = (float)shift - (m == -INFINITY ? 0.0f : m);
                        float sum[2] = {0.0f, 0.0f};
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = ex2(fmaf(__uint_as_float(r[2 * i]), f, less)), y = ex2(fmaf(__uint_as_float(r[2 * i + 1]), f, less));
                            sum[0] += x;
                            sum[1] += y;
                            w[i] = half2_bits(x, y);
                        }
                        l = fmaf(sum[0] + sum[1], pow2(-shift), l);
                        tmem_store16(at_s + 16 * c, w);
                    }
                    ev = new_ev;
                    tmem_stored();
                }
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar_p + 8 * grp);
                const ChunkMeta& meta = s_meta[step & 3u];
                const uint4 any = *reinterpret_cast<const uint4*>(meta.any_poison);
                if (any.x | any.y | any.z | any.w) {
                    const int tok0 = (g.t.from + g.c0 + j) * kChunkStep;
                    for (int i = 0; i < NG; ++i)
                        for (int c = 0; c < 4; ++c)
                            for (uint32_t bits = meta.poison[i][c]; bits; bits &= bits - 1u) {
                                const int at = tok0 + 32 * c + __ffs(bits) - 1;
                                if (at >= from && at < to) bad |= 1u << i;
                            }
                }
            }
            bar_wait(bar_o, seg & 1u, gave_up, p.err);
            ++seg;
            tc_after();
            const bool whole = g.c0 == 0 && g.c1 == g.t.steps, late = g.c0 > 0;
            if (active && any_live) {
                const long long tok = g.r.start + query, qh = (long long)g.head * p.ratio + sub;
                float* part = p.part + ((size_t)blockIdx.x * 2u + (late ? 0u : 1u)) * kv4_part_floats(D, kChunkRows / 8);
                const float unit = pow2(min(max(ev - 12, -126), 127)), by = whole ? (l == 0.0f ? 0.0f : unit / l) : unit;
                T* dst = reinterpret_cast<T*>(p.out) + tok * p.out_token + qh * p.out_head;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t r[32];
                    tmem_load32(at_o + 32 * c, r);
                    tmem_loaded();
                    if (live) {
                        const float nan = __int_as_float(0x7fc00000);
                        const bool is_bad = (bad >> (32 * c / GS)) & 1u;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float o[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[i] = is_bad ? nan : __uint_as_float(r[8 * i + e]) * by;
                            if (whole) *reinterpret_cast<uint2*>(dst + 32 * c + 4 * e) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
                            else __stcg(reinterpret_cast<float4*>(part + row * D + 32 * c + 4 * e), make_float4(o[0], o[1], o[2], o[3]));
                        }
                    }
                }
                if (live) {
                    if (!whole) {
                        part[kChunkRows * D + 2 * row] = m;
                        part[kChunkRows * D + 2 * row + 1] = l;
                    } else if (p.lse) {
                        p.lse[(size_t)tok * p.kv_heads * p.ratio + qh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
                    }
                }
            }
            tc_before();
            if (!whole && !late && row == 0) {
                cut.parts = (uint32_t)(ratio_of(g.x - g.pos + g.t.steps + kSegmentSteps - 1, per) - blockIdx.x) + 1u;
                cut.row0 = (uint32_t)(g.t.q0 * (int)p.ratio); cut.head = (uint32_t)g.head; cut.start = (uint32_t)g.r.start;
                cut.rows = (uint32_t)((g.t.q0 + g.t.n) * (int)p.ratio);
            }
        }
        if (row == 0) reinterpret_cast<Kv4Cut*>(p.part + (size_t)gridDim.x * 2u * kv4_part_floats(D, kChunkRows / 8))[blockIdx.x] = cut;
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---- launch ------------------------------------------------------------------------------------------------
template <int D, int GS, int DT> cudaError_t run_chunk(const Kv4Attn& p, uint32_t blocks, cudaStream_t s) {
    static bool ready[64] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!ready[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(kv4_chunk_kernel<D, GS, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ChunkShape<D>::kBytes)) return e;
        ready[dev] = true;
    }
    if (cudaError_t e = launch_early(kv4_chunk_kernel<D, GS, DT>, dim3(blocks), dim3(kChunkThreads), ChunkShape<D>::kBytes, s, p)) return e;
    return launch_early(kv4_join_kernel<D, kChunkRows / 8, DT>, dim3(blocks, 8), dim3(JoinShape<D>::kThreads), 0, s, p, blocks);
}

}  // namespace dd
