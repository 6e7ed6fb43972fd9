// Attention of a few queries over the 4-bit cache (decoding, drafted tokens).
//
// softmax(q k^T s) v with k, v = middle + step * (code - 8), middle = offset + 8 step, never formed: with c = code - 8 as tensor-core
// factors
//   scores      q.k = sum_g step_g (q_g . c_g) + middle_g (1 . q_g)                per token and group g of the head
//   outputs     p v = sum_t (p_t step_t) c_t + sum_t p_t middle_t
// so the codes are the only operands made from the cache: a mask and an OR turn two codes of a word into fp16 numbers 1024 + code (or
// 1024 + 16 code), one fused multiply-add into code - 8, exact.  (The masked word alone is a pair of subnormal fp16 numbers code * 2^-24
// and would save that instruction, but the tensor cores align subnormal products ten bits too high: scores lost 2^-14 of their terms.  And
// codes of one sign make sums that grow with the context and are cut off in one direction at every step.)  Tokens are the 16 rows of
// an operand in the scores (m16n8k16, 8 queries wide) and its depth in the outputs, so a batch-1 token with 4 queries per key head
// fills half of each instruction instead of a quarter.
//   queries     fp16 after scaling each row to a power of two near 2^9: exact for both 16-bit types (elements below 2^-23 of the row's
//               largest lose bits)
//   weights     p_t * step_t in fp16 with the steps scaled by a running power of two per group, so that neither small steps nor
//               small weights become subnormal before they are 2^-23 of the largest (the largest step of the cells that the warp has
//               met, seen by the row or not)
//   the rest    (scores, running maximum and sum, the middles' part, sums over thread blocks) in fp32
//
// A step of two cells takes a warp 2340 cycles, 390 a cell of 2176 bytes (heads of 128, one group) and scheduler, where the copy rate allows
// 354; then come the ends of segments.  Neither is full under the profiler: memory 45 %, issue slots 48 %.  64 requests of 512 to 16384 tokens,
// 372 MB: 84 to 90 us, 4.1 to 4.4 TB/s.
//
// The work is a line of cells (16 tokens of one key head), request by request, and every thread block takes an equal part of it
// (lengths are on the device: each block sums them itself); work that would not fill the device is cut by segments instead.  A warp streams
// its own cells through shared memory (cp.async, kStages steps ahead) and keeps its own running maximum and sums; the four warps of a block are added where a segment (one request, head and
// tile of 8 or 16 query rows) ends.  A segment that blocks share leaves its parts in `part`, and kv4_join adds them.
#pragma once
#include "kv4.cuh"

namespace dd {

constexpr int kDecodeThreads = 128;
constexpr int kDecodeWarps = 4;
constexpr uint32_t kNoCell = 0xffffffffu;
constexpr float kGrow = 4.0f;          // a running maximum follows once it is 2^4 behind
// Factors of the scores stay above 0, where a hidden score of -inf would become NaN.  A score is then off by 2^-104 times the largest element
// of the keys here (sums of 256 products with queries below 2^14), by 2^-92 in the tiles, whose keys are scaled too.
constexpr float kLeastFactor = 1.17549435e-38f;

// one part of a cut segment: [rows of a tile][D] sums, then [rows][2] maximum (log2 units) and sum
__host__ __device__ constexpr uint32_t kv4_part_floats(uint32_t d, uint32_t nt) { return 8u * nt * (d + 2u); }

// how many parts, and of which segment, the block that began a cut segment leaves behind
struct Kv4Cut {
    uint32_t parts;                    // 0: this block cut no segment that it began
    uint32_t row0, head;               // row0: first row of the tile among the request's rows
    uint32_t start, rows;              // first token of the request among all, rows of the request
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 bytes into shared memory, zeros where `bytes` is 0
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }     // -126 <= e <= 127

// the larger of each 16-bit pair, the number where one is NaN
template <int DT> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (DT == FP16) {
        const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// the codes of a word less 8, as fp16 pairs: (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void code_pairs(uint32_t x, uint32_t (&h)[4]) {
    const __half2 low = __float2half2_rn(-1032.0f), by = __float2half2_rn(0.0625f), high = __float2half2_rn(-72.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = i < 2 ? x : x >> 8;
        uint32_t m;                                          // (y & mask) | 0x64006400 as one instruction
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(y), "r"(i & 1 ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
        const __half2 v = *reinterpret_cast<const __half2*>(&m);
        const __half2 r = i & 1 ? __hfma2(v, by, high) : __hadd2(v, low);
        h[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
}

// the codes of a word as fp16 pairs 1024 + 16 code: (0, 4), (1, 5), (2, 6), (3, 7).  Two instructions a pair less than above; the 1024 is
// taken out of the sums over a head, which costs them 2^-21 of their terms.
__device__ __forceinline__ void raised_pairs(uint32_t x, uint32_t (&h)[4]) {
    const __half2 by = __float2half2_rn(16.0f), less = __float2half2_rn(-15360.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = i < 2 ? x : x >> 8;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(h[i]) : "r"(y), "r"(i & 1 ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
        if (!(i & 1)) {
            const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&h[i]), by, less);       // 16 (1024 + code) - 15 * 1024
            h[i] = *reinterpret_cast<const uint32_t*>(&r);
        }
    }
}

// N consecutive 32-bit words of shared memory, in the widest loads
template <int N> __device__ __forceinline__ void load_words(uint32_t (&x)[N], const uint8_t* at) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(at + 4 * i);
            x[i] = u.x; x[i + 1] = u.y; x[i + 2] = u.z; x[i + 3] = u.w;
        }
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(at);
        x[0] = u.x; x[1] = u.y;
    } else {
        x[0] = *reinterpret_cast<const uint32_t*>(at);
    }
}

// quotient of numbers that almost always fit 32 bits, where a division costs a fifth
__device__ __forceinline__ unsigned long long ratio_of(unsigned long long a, unsigned long long b) {
    return ((a | b) >> 32) == 0 ? (unsigned long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// what a request asks for
struct Kv4Request {
    int start, queries, length;        // first row, rows, tokens in the cache
    int first, cells;                  // cells that some query sees: first, number (at least one)
    int tiles;                         // tiles of query rows
};

__device__ __forceinline__ Kv4Request kv4_request(const Kv4Attn& p, uint32_t b, int tile_rows, bool report) {
    Kv4Request r;
    const int rows = (int)p.rows;
    r.start = min(max(p.starts[b], 0), rows);
    r.queries = max(min(max(p.starts[b + 1], 0), rows) - r.start, 0);
    r.length = max(p.lengths[b], 0);
    const long long most = (long long)p.table_cols * p.page_cells * kCellTokens;
    if ((long long)r.length > most) {
        if (report) raise_error(p.err, kErrKv4Page);
        r.length = (int)most;
    }
    r.first = p.window ? max(0ll, (long long)r.length - r.queries - (long long)p.window + 1) / kCellTokens : 0;
    r.cells = max(1, (r.length + kCellTokens - 1) / kCellTokens - r.first);
    r.tiles = (int)(((long long)r.queries * p.ratio + tile_rows - 1) / tile_rows);
    return r;
}

// Pieces of a segment where each has a block to itself: one up to 16 cells (two steps of a warp; a step costs 0.8 us, a join 2), then of 8
// cells.  One request with 8 key heads, this / blocks of 8 cells cut from the line (us): 16 tokens 6.9 / 31 (one block has all heads), 100 tokens
// 7.3 / 11.4, 777 tokens 9.7 / 12.5, 3000 tokens 10.3 / 12.9 (heads of 128).
__host__ __device__ constexpr int kv4_pieces(int cells) { return cells <= 16 ? 1 : (cells + 7) / 8; }

// What the beginning and the end of a segment (queries, first cells, adding the warps' sums) cost a block, in cells: 5 to 10 thousand cycles
// at 290 a cell.  Counted as 0 / 16 / 32 / 48 cells: 64 requests of 512 to 16384 tokens 112 / 93 / 84 / 86 us, drafts of 17 requests 104 / 69 / 61
// / 63: without it the blocks that have the short requests take twice as long as the others.  Measured with heads of 128; one number for all, though
// a cell of a head of 64 costs about half as much, one of 256 twice.
constexpr int kSegmentCells = 32;

// the rows before the first request and behind the last, a row a block at a time
template <int D, int DT> __device__ __forceinline__ void clear_rest(const Kv4Attn& p, int tid, int threads) {
    using T = typename Tr<DT>::T;
    const int rows = (int)p.rows, first = p.requests ? min(max(p.starts[0], 0), rows) : 0, end = p.requests ? min(max(p.starts[p.requests], 0), rows) : 0;
    for (long long i = blockIdx.x; i < (long long)first + (rows - end); i += gridDim.x) {
        const int t = i < first ? (int)i : end + (int)(i - first);
        for (uint32_t e = tid; e < p.kv_heads * p.ratio * D; e += threads)
            reinterpret_cast<T*>(p.out)[(long long)t * p.out_token + (long long)(e / D) * p.out_head + e % D] = Tr<DT>::from_f(0.0f);
        if (p.lse)
            for (uint32_t e = tid; e < p.kv_heads * p.ratio; e += threads) p.lse[(size_t)t * p.kv_heads * p.ratio + e] = -INFINITY;
    }
}

template <int D, int NT> struct DecodeShape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kRowStride = D + 4;            // floats; keeps the warps' 16-byte stores apart by banks
    static constexpr int kMergeFloats = kDecodeWarps * kRows * (kRowStride + 2);
};
// A step of a warp is two neighbouring cells (32 tokens), and kStages steps of a warp lie in shared memory, beside the place where the
// warps' sums are added: the next segment's first steps are under way meanwhile.
constexpr int kStages = 3, kCells = 2;
template <int D, int GS, int NT> __host__ __device__ constexpr size_t decode_smem() {
    return (size_t)kDecodeWarps * kStages * (uint32_t)kCells * kv4_cell_bytes(D, GS) + DecodeShape<D, NT>::kMergeFloats * 4u;
}

// blocks of an SM that the registers are cut for: as many as need no spills worth the name
template <int D, int GS, int NT> __host__ __device__ constexpr int decode_residency() {
    return D == 256 ? 2 : NT == 1 ? (D == 64 ? 4 : 3) : D == 64 ? 3 : 2;
}

template <int D, int GS, int NT, int DT>
__global__ void __launch_bounds__(kDecodeThreads, decode_residency<D, GS, NT>()) kv4_decode_kernel(Kv4Attn p) {
    using T = typename Tr<DT>::T;
    using Sh = DecodeShape<D, NT>;
    constexpr int NG = D / GS;                  // groups of a head
    constexpr int NW = D / 32;                  // words of 32 elements
    constexpr uint32_t CELL = kv4_cell_bytes(D, GS);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_sum[2][kDecodeThreads / 32];
    __shared__ long long s_rest;
    __shared__ uint32_t s_request;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gid = lane >> 2, tig = lane & 3;
    uint8_t* ring = smem + (size_t)warp * kStages * kCells * CELL;
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    float* merge = reinterpret_cast<float*>(smem + (size_t)kDecodeWarps * kStages * kCells * CELL);   // [warp][row][kRowStride]
    float* merge_ml = merge + kDecodeWarps * Sh::kRows * Sh::kRowStride;                      // [warp][row][2]
    uint8_t* after = reinterpret_cast<uint8_t*>(p.part + (size_t)gridDim.x * 2u * kv4_part_floats(D, NT));
    Kv4Cut* cuts = reinterpret_cast<Kv4Cut*>(after);

    pdl_trigger();
    pdl_wait();

    // ---- this block's part of the line of cells; or, while there are blocks for every segment or piece of one, a segment or a piece
    const uint32_t run = (p.requests + kDecodeThreads - 1u) / kDecodeThreads;
    const uint32_t rb0 = min(tid * run, p.requests), rb1 = min(rb0 + run, p.requests);
    long long mine[2] = {0, 0};                                // cells, pieces
    for (uint32_t b = rb0; b < rb1; ++b) {
        const Kv4Request r = kv4_request(p, b, Sh::kRows, blockIdx.x == 0);
        mine[0] += (long long)r.tiles * p.kv_heads * (r.cells + kSegmentCells);
        mine[1] += (long long)r.tiles * p.kv_heads * kv4_pieces(r.cells);
    }
    long long incl[2] = {mine[0], mine[1]};
#pragma unroll
    for (int o = 1; o < 32; o *= 2)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long long n = __shfl_up_sync(0xffffffffu, incl[i], o);
            if (lane >= o) incl[i] += n;
        }
    if (lane == 31) { s_sum[0][warp] = incl[0]; s_sum[1][warp] = incl[1]; }
    __syncthreads();
    long long before[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (w < warp) before[i] += s_sum[i][w];
            all[i] += s_sum[i][w];
        }
    const bool pieces = all[1] <= (long long)gridDim.x;
    const int kind = pieces ? 1 : 0;
    const long long total = pieces ? all[1] : all[0];
    // at least two cells a warp: a shorter part would spend its time in the joining of the parts
    const long long per = pieces ? 1 : max((long long)ratio_of(total + gridDim.x - 1, gridDim.x), 2ll * kDecodeWarps);
    const long long at0 = (long long)blockIdx.x * per;
    long long x0 = at0, x1 = min(at0 + per, total);
    {
        const long long excl = (pieces ? before[1] + incl[1] - mine[1] : before[0] + incl[0] - mine[0]), own = pieces ? mine[1] : mine[0];
        if (x0 < x1 && excl <= x0 && x0 < excl + own) {
            long long at = excl;
            uint32_t b = rb0;
            for (;; ++b) {                                   // ends: x0 lies below the end of this run
                const Kv4Request r = kv4_request(p, b, Sh::kRows, false);
                const long long n = (long long)r.tiles * p.kv_heads * (kind ? kv4_pieces(r.cells) : r.cells + kSegmentCells);
                if (x0 < at + n) break;
                at += n;
            }
            s_request = b;
            s_rest = x0 - at;
        }
    }
    __syncthreads();
    if (p.clear_rest) clear_rest<D, DT>(p, tid, kDecodeThreads);
    Kv4Cut cut = {};
    if (x0 < x1) {
        uint32_t b = s_request;
        Kv4Request rq = kv4_request(p, b, Sh::kRows, false);
        int unit = pieces ? kv4_pieces(rq.cells) : rq.cells + kSegmentCells;
        int item = (int)ratio_of(s_rest, unit);              // tile * kv_heads + head
        int pos = (int)(s_rest - (long long)item * unit);    // in the segment's part of the line: kSegmentCells for its beginning and end, its cells
        uint32_t head = (uint32_t)item % p.kv_heads;
        long long x = x0;
        int take, c0, c1;                                    // of the line; cells
        auto range = [&] {
            take = (int)min((long long)(unit - pos), x1 - x);
            c0 = pieces ? (int)((long long)pos * rq.cells / unit) : max(pos - kSegmentCells, 0);
            c1 = pieces ? (int)((long long)(pos + take) * rq.cells / unit) : max(pos + take - kSegmentCells, 0);
        };
        range();

        // ---- this warp's steps of a segment: cells c0 + 2 (warp + 4 j), + 1
        int count;
        uint32_t cell_at, fill;                              // place in the cache of the cell 2 j + lane of its steps; stage that is filled next
        auto places_of = [&](int j0) {
            const int c = rq.first + c0 + kCells * (warp + kDecodeWarps * (j0 + lane / kCells)) + lane % kCells;
            cell_at = kNoCell;
            if (c < rq.first + c1 && c * kCellTokens < rq.length) {
                const uint32_t column = (uint32_t)c / p.page_cells;
                const int page = p.table[(long long)b * p.table_stride + column];
                if (page >= 0 && (uint32_t)page < p.pages) cell_at = ((uint32_t)page * p.kv_heads + head) * p.page_cells + (uint32_t)c % p.page_cells;
                else raise_error(p.err, kErrKv4Page);
            }
        };
        auto issue = [&](int j) {
            if (j < count) {
                if (j % (32 / kCells) == 0) places_of(j);
#pragma unroll
                for (int u = 0; u < kCells; ++u) {
                    const uint32_t at = __shfl_sync(0xffffffffu, cell_at, kCells * (j % (32 / kCells)) + u);
                    const uint32_t bytes = at == kNoCell ? 0u : 16u;       // zeros, from a source that is not read
                    const uint8_t* src = p.cache + (size_t)(at == kNoCell ? 0u : at) * CELL + lane * 16u;
#pragma unroll
                    for (uint32_t i = 0; i < (CELL / 16 + 31) / 32; ++i)
                        if (CELL % 512 == 0 || i * 512u + lane * 16u < CELL) cp_async16(fill + u * CELL + i * 512u, src + i * 512u, bytes);
                }
                fill = fill == ring_s + lane * 16u + (kStages - 1u) * kCells * CELL ? ring_s + lane * 16u : fill + kCells * CELL;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto begin = [&] {
            count = ((c1 - c0 + kCells - 1) / kCells - warp + kDecodeWarps - 1) / kDecodeWarps;
            fill = ring_s + lane * 16u;
#pragma unroll
            for (int j = 0; j < kStages - 1; ++j) issue(j);
        };
        if (c1 > c0) begin();
        while (x < x1 && c1 > c0) {                          // a range that ends before the first cell of its last segment leaves that to the next
            const int row0 = (int)((uint32_t)item / p.kv_heads) * Sh::kRows;
            const int all_rows = rq.queries * (int)p.ratio;

            // ---- queries of the tile as operands: lane (gid, tig) holds row gid, elements 32 w + 8 tig .. + 7
            uint32_t qf[NT][NW][4];                          // pairs (0,4), (1,5), (2,6), (3,7)
            float sf[NT][2], qs[NT][2][NG];                  // of the rows 2 tig, 2 tig + 1 that this lane meets in the sums
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = row0 + 8 * nt + gid;
                const bool live = row < all_rows;
                const int tok = rq.start + (live ? row / (int)p.ratio : 0);
                const T* src = reinterpret_cast<const T*>(p.q.p) + (long long)tok * p.q.token + (long long)(head * p.ratio + (live ? row % (int)p.ratio : 0)) * p.q.head;
                float v[NW][8];
                float most = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    uint4 raw = make_uint4(0, 0, 0, 0);
                    if (live) {
                        if (p.q_vec) {
                            raw = *reinterpret_cast<const uint4*>(src + 32 * w + 8 * tig);
                        } else {
                            uint32_t u[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint16_t* e = reinterpret_cast<const uint16_t*>(src + 32 * w + 8 * tig + 2 * i);
                                u[i] = (uint32_t)e[0] | (uint32_t)e[1] << 16;
                            }
                            raw = make_uint4(u[0], u[1], u[2], u[3]);
                        }
                    }
                    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = unpack2<DT>(u[i]);
                        v[w][2 * i] = f.x;
                        v[w][2 * i + 1] = f.y;
                        most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                int e = (int)(__float_as_uint(most) >> 23) - 127;      // the row's exponent
                e = (most > 0.0f && most < INFINITY) ? max(e, -87) : 9;
                const float up = pow2(9 - e);                          // and the raised codes bring 2^4
                float sum[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) sum[g] = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[w][i] *= up;
                        sum[w * 32 / GS] += v[w][i];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[nt][w][i] = half2_bits(v[w][i], v[w][i + 4]);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
                    sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
                    sum[g] *= 16.0f;
                }
                const float mine_sf = fmaxf(p.scale_log2 * pow2(e - 13), kLeastFactor);      // the sums with codes are 16 times too large
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    sf[nt][i] = __shfl_sync(0xffffffffu, mine_sf, 8 * tig + 4 * i);
#pragma unroll
                    for (int g = 0; g < NG; ++g) qs[nt][i][g] = __shfl_sync(0xffffffffu, sum[g], 8 * tig + 4 * i);
                }
            }
            // tokens that each of this lane's rows sees: [from, to)
            int from[NT][2], to[NT][2];
            const int pos0 = rq.length - rq.queries, end = (rq.first + c1) * kCellTokens;        // the segment's cells end there
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = row0 + 8 * nt + 2 * tig + i;
                    const int pos = pos0 + min(row, all_rows - 1) / (int)p.ratio;
                    to[nt][i] = min(max(pos + 1, 0), end);
                    from[nt][i] = p.window ? (int)max(0ll, (long long)pos - (long long)p.window + 1) : 0;
                }
            // cells between these are seen whole by every row of the tile
            const int first_pos = pos0 + row0 / (int)p.ratio, last_pos = pos0 + (min(row0 + Sh::kRows, all_rows) - 1) / (int)p.ratio;
            const int clear_to = min(max(first_pos + 1, 0), end), clear_from = p.window ? (int)max(0ll, (long long)last_pos - (long long)p.window + 1) : 0;

            float acc[D / 16][NT][4], off[NT][2][NG], l[NT][2], m[NT][2], less[NT][2];
            float fv[NG], limit[NG];                         // factor of the steps, and the step that it is good for
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][nt][j] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                fv[g] = 0.0f;
                limit[g] = -1.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) off[nt][0][g] = off[nt][1][g] = 0.0f;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) { l[nt][i] = 0.0f; m[nt][i] = -INFINITY; less[nt][i] = 0.0f; }

            // One step.  clear: every row of the tile sees all 32 tokens.
            auto step = [&](const uint8_t* st, int tok0, bool clear) {
                constexpr int PER = NW < 4 ? NW : 4;          // words of a lane in a block
                constexpr int VB = D < 128 ? 1 : D / 128, VP = NW / VB;      // blocks of values, words of a lane and plane in each
                // ---- scores: rows = tokens gid, gid + 8 of cell u; columns = queries 2 tig, 2 tig + 1
                float s[kCells][NT][4];
                uint32_t vr[kCells][2][NG];                        // steps and offsets of the values
#pragma unroll
                for (int u = 0; u < kCells; ++u) {
                    const uint8_t* cell = st + u * CELL;
                    uint32_t kr[2][NG];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        load_words(kr[i], cell + kv4_key_step(D, GS, gid + 8 * i, 0));
                        load_words(vr[u][i], cell + kv4_value_step(D, GS, gid + 8 * i, 0));
                    }
                    uint32_t xa[NW / PER][PER], xb[NW / PER][PER];
#pragma unroll
                    for (int bl = 0; bl < NW / PER; ++bl) {
                        load_words(xa[bl], cell + ((bl * 16 + gid) * 4 + tig) * PER * 4);
                        load_words(xb[bl], cell + ((bl * 16 + gid + 8) * 4 + tig) * PER * 4);
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float raw[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) raw[nt][i] = 0.0f;
#pragma unroll
                        for (int w = g * GS / 32; w < (g + 1) * GS / 32; ++w) {
                            uint32_t ca[4], cb[4];
                            raised_pairs(xa[w / PER][w % PER], ca);
                            raised_pairs(xb[w / PER][w % PER], cb);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma_16816<FP16>(raw[nt], ca[0], cb[0], ca[1], cb[1], qf[nt][w][0], qf[nt][w][1]);
                                mma_16816<FP16>(raw[nt], ca[2], cb[2], ca[3], cb[3], qf[nt][w][2], qf[nt][w][3]);
                            }
                        }
                        float ks[2], ko[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float2 f = unpack2<DT>(kr[i][g]);
                            ks[i] = f.x;
                            ko[i] = fmaf(-64.0f, f.x, f.y);            // offset less the 1024 / 16 steps that the codes are raised by
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float middle = ko[i >> 1] * qs[nt][i & 1][g];
                                s[u][nt][i] = fmaf(raw[nt][i], ks[i >> 1], g == 0 ? middle : s[u][nt][i] + middle);
                            }
                    }
                }
                bool poison = false;                          // a token that some row does not see holds no number: its product with 0 counts
                if (!clear) {
#pragma unroll
                    for (int u = 0; u < kCells; ++u) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int tok = tok0 + 16 * u + gid + 8 * (i >> 1);
                                if (tok < from[nt][i & 1] || tok >= to[nt][i & 1]) s[u][nt][i] = -INFINITY;
                            }
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int g = 0; g < NG; ++g) {
                                if (tok0 + 16 * u + 8 * i + gid >= rq.length) vr[u][i][g] = 0u;      // behind the end lies what the page held before
                                poison |= !(fabsf(unpack2<DT>(vr[u][i][g]).y) < INFINITY);
                            }
                    }
                    poison = __any_sync(0xffffffffu, poison);
                }
                // the step's largest scores and steps of the values
                float high[NT][2], steps[NG];
                bool follow = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(s[0][nt][i], s[0][nt][2 + i]);
#pragma unroll
                        for (int u = 1; u < kCells; ++u) top = fmaxf(top, fmaxf(s[u][nt][i], s[u][nt][2 + i]));
                        high[nt][i] = top * sf[nt][i];
                        follow |= high[nt][i] > m[nt][i] + kGrow;
                    }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    uint32_t top = max2<DT>(vr[0][0][g], vr[0][1][g]);
#pragma unroll
                    for (int u = 1; u < kCells; ++u) top = max2<DT>(top, max2<DT>(vr[u][0][g], vr[u][1][g]));
                    steps[g] = unpack2<DT>(top).x;
                    follow |= steps[g] > limit[g];
                }
                if (__any_sync(0xffffffffu, follow)) {
                    // maxima over the step, sums brought to them; rare once a few cells are done
                    float down[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float top = high[nt][i];
#pragma unroll
                            for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            top = fmaxf(top, m[nt][i]);
                            down[nt][i] = top == m[nt][i] ? 1.0f : ex2(m[nt][i] - top);
                            m[nt][i] = top;
                            less[nt][i] = top == -INFINITY ? 0.0f : top;      // a row that has seen nothing yet: its weights are 0
                            l[nt][i] *= down[nt][i];
                        }
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(steps[g], 0.0f)));
                        const int e = min(max((int)(bits >> 23) - 127, -100), 127);   // the largest step is below 2^(e+1)
                        const float want = pow2(10 - e);
                        float by = 1.0f;
                        if (limit[g] < 0.0f || want < fv[g]) {
                            by = limit[g] < 0.0f ? 0.0f : want / fv[g];               // the sums are still 0 at first
                            fv[g] = want;
                            limit[g] = pow2(e + 1);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float d0 = by * down[nt][0], d1 = by * down[nt][1];
                            off[nt][0][g] *= down[nt][0];
                            off[nt][1][g] *= down[nt][1];
#pragma unroll
                            for (int i = g * GS / 16; i < (g + 1) * GS / 16; ++i) {
                                acc[i][nt][0] *= d0; acc[i][nt][1] *= d1; acc[i][nt][2] *= d0; acc[i][nt][3] *= d1;
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < kCells; ++u) {
                    const uint8_t* cell = st + u * CELL;
                    float w[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[nt][i] = ex2(fmaf(s[u][nt][i], sf[nt][i & 1], -less[nt][i & 1]));
                            l[nt][i & 1] += w[nt][i];
                        }
                    // ---- outputs: rows = elements, depth = tokens, columns = queries; planes of tokens 0..7 and 8..15
                    uint32_t xv[VB][2][VP];
#pragma unroll
                    for (int bl = 0; bl < VB; ++bl)
#pragma unroll
                        for (int c = 0; c < 2; ++c) load_words(xv[bl][c], cell + 8 * D + ((bl * 2 + c) * 32 + lane) * (VP * 4));
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        uint32_t b0[NT], b1[NT];
                        const float2 v0 = unpack2<DT>(vr[u][0][g]), v1 = unpack2<DT>(vr[u][1][g]);
                        const float f0 = v0.x * fv[g], f1 = v1.x * fv[g], o0 = fmaf(8.0f, v0.x, v0.y), o1 = fmaf(8.0f, v1.x, v1.y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            b0[nt] = movmatrix(half2_bits(w[nt][0] * f0, w[nt][1] * f0));
                            b1[nt] = movmatrix(half2_bits(w[nt][2] * f1, w[nt][3] * f1));
                            if (!poison) {
#pragma unroll
                                for (int i = 0; i < 2; ++i) off[nt][i][g] = fmaf(w[nt][i], o0, fmaf(w[nt][2 + i], o1, off[nt][i][g]));
                            } else {
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    off[nt][i][g] += w[nt][i] == 0.0f ? 0.0f : w[nt][i] * o0;
                                    off[nt][i][g] += w[nt][2 + i] == 0.0f ? 0.0f : w[nt][2 + i] * o1;
                                }
                            }
                        }
#pragma unroll
                        for (int i = g * GS / 32; i < (g + 1) * GS / 32; ++i) {      // elements 32 i .. + 31, four of them in the lane's word
                            uint32_t c0v[4], c1v[4];
                            code_pairs(xv[i / VP][0][i % VP], c0v);
                            code_pairs(xv[i / VP][1][i % VP], c1v);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma_16816<FP16>(acc[2 * i][nt], c0v[0], c0v[1], c1v[0], c1v[1], b0[nt], b1[nt]);
                                mma_16816<FP16>(acc[2 * i + 1][nt], c0v[2], c0v[3], c1v[2], c1v[3], b0[nt], b1[nt]);
                            }
                        }
                    }
                }
            };
            const uint8_t* st = ring;
            int tok0 = (rq.first + c0 + kCells * warp) * kCellTokens;
            for (int j = 0; j < count; ++j) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
                __syncwarp();
                issue(j + kStages - 1);                      // into the stage that the last step read
                // behind the end of the segment's cells lies another block's work: `to` hides it
                step(st, tok0, tok0 >= clear_from && tok0 + kCells * kCellTokens <= clear_to);
                st = st == ring + (kStages - 1) * kCells * CELL ? ring : st + kCells * CELL;
                tok0 += kDecodeWarps * kCells * kCellTokens;
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();                                    // the warp is through with its ring

            // ---- on to the next segment, whose first steps travel while this one's sums are added
            const bool whole = c0 == 0 && c1 == rq.cells, late = c0 > 0;
            const int start = rq.start;
            const uint32_t at_head = head;
            if (!whole && !late) {                           // it ends in the block that has the segment's last place on the line
                cut.parts = pieces ? (uint32_t)kv4_pieces(rq.cells) : (uint32_t)(ratio_of(x - pos + unit - 1, per) - blockIdx.x) + 1u;
                cut.row0 = (uint32_t)row0; cut.head = head; cut.start = (uint32_t)start; cut.rows = (uint32_t)all_rows;
            }
            x += take;
            if (x < x1) {
                if (++item == rq.tiles * (int)p.kv_heads) {
                    item = 0;
                    do rq = kv4_request(p, ++b, Sh::kRows, false); while (rq.tiles == 0);      // ends: cells remain
                }
                unit = rq.cells + kSegmentCells;             // a piece is a block's only one
                pos = 0;
                head = (uint32_t)item % p.kv_heads;
                range();
                if (c1 > c0) begin();
            }

            // ---- the warps' sums into shared memory
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int o = 4; o < 32; o *= 2) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], o);
                    const int row = 8 * nt + 2 * tig + i;
                    if (gid == 0) {
                        merge_ml[(warp * Sh::kRows + row) * 2] = m[nt][i];
                        merge_ml[(warp * Sh::kRows + row) * 2 + 1] = l[nt][i];
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float o4 = off[nt][i][g];
#pragma unroll
                        for (int o = 4; o < 32; o *= 2) o4 += __shfl_xor_sync(0xffffffffu, o4, o);
                        const float unit = fv[g] != 0.0f ? 1.0f / fv[g] : 0.0f;
#pragma unroll
                        for (int k = g * GS / 32; k < (g + 1) * GS / 32; ++k) {
                            float4 v;
                            v.x = fmaf(acc[2 * k][nt][i], unit, o4);
                            v.y = fmaf(acc[2 * k][nt][2 + i], unit, o4);
                            v.z = fmaf(acc[2 * k + 1][nt][i], unit, o4);
                            v.w = fmaf(acc[2 * k + 1][nt][2 + i], unit, o4);
                            *reinterpret_cast<float4*>(merge + (size_t)(warp * Sh::kRows + row) * Sh::kRowStride + 32 * k + 4 * gid) = v;
                        }
                    }
                }
            __syncthreads();
            float* part = p.part + ((size_t)blockIdx.x * 2u + (late ? 0u : 1u)) * kv4_part_floats(D, NT);
            for (int e = tid; e < Sh::kRows * (D / 4); e += kDecodeThreads) {
                const int r = e / (D / 4), d4 = e % (D / 4);
                float top = -INFINITY, mw[kDecodeWarps];
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) {
                    mw[w] = merge_ml[(w * Sh::kRows + r) * 2];
                    top = fmaxf(top, mw[w]);
                }
                float sum = 0.0f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) {
                    if (mw[w] == -INFINITY && merge_ml[(w * Sh::kRows + r) * 2 + 1] == 0.0f) continue;       // saw nothing
                    const float f = mw[w] == top ? 1.0f : ex2(mw[w] - top);
                    const float4 o = *reinterpret_cast<const float4*>(merge + (size_t)(w * Sh::kRows + r) * Sh::kRowStride + 4 * d4);
                    sum = fmaf(merge_ml[(w * Sh::kRows + r) * 2 + 1], f, sum);
                    v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
                }
                const int row = row0 + r;
                if (whole) {
                    if (row < all_rows) {
                        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                        const long long tok = start + row / (int)p.ratio, h = at_head * p.ratio + row % (int)p.ratio;
                        T* dst = reinterpret_cast<T*>(p.out) + tok * p.out_token + h * p.out_head + 4 * d4;
                        T o[4] = {Tr<DT>::from_f(v.x * inv), Tr<DT>::from_f(v.y * inv), Tr<DT>::from_f(v.z * inv), Tr<DT>::from_f(v.w * inv)};
                        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
                        if (p.lse && d4 == 0) p.lse[(size_t)tok * p.kv_heads * p.ratio + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
                    }
                } else {
                    __stcg(reinterpret_cast<float4*>(part + r * D + 4 * d4), v);
                    if (d4 == 0) {
                        part[Sh::kRows * D + 2 * r] = top;
                        part[Sh::kRows * D + 2 * r + 1] = sum;
                    }
                }
            }
            __syncthreads();
        }
    }
    if (tid == 0) cuts[blockIdx.x] = cut;
}

// Adds the parts of a cut segment: a block takes four rows of it, and four parts of a row at the same time (two for heads of 256).  Few
// blocks, since most cut segments have two or three parts and a block waits three round trips for them: one block a row took 30 us behind
// 64 requests.
constexpr int kJoinRows = 4;
template <int D> struct JoinShape {
    static constexpr int kLanes = D / 4, kWays = D == 256 ? 2 : 4, kThreads = kLanes * kWays * kJoinRows;
};

template <int D, int NT, int DT>
__global__ void __launch_bounds__(JoinShape<D>::kThreads) kv4_join_kernel(Kv4Attn p, uint32_t blocks) {
    using T = typename Tr<DT>::T;
    constexpr uint32_t LANES = JoinShape<D>::kLanes, WAYS = JoinShape<D>::kWays;
    __shared__ float4 s_v[kJoinRows][WAYS][LANES];
    __shared__ float s_ml[kJoinRows][WAYS][2];
    pdl_trigger();
    pdl_wait();
    const Kv4Cut cut = reinterpret_cast<const Kv4Cut*>(p.part + (size_t)blocks * 2u * kv4_part_floats(D, NT))[blockIdx.x];
    if (cut.parts == 0) return;
    const float* base = p.part + (size_t)blockIdx.x * 2u * kv4_part_floats(D, NT);
    const uint32_t d4 = threadIdx.x % LANES, way = threadIdx.x / LANES % WAYS, mine = threadIdx.x / (LANES * WAYS);
    for (uint32_t r0 = blockIdx.y * kJoinRows; r0 < 8 * NT && cut.row0 + r0 < cut.rows; r0 += gridDim.y * kJoinRows) {
        const uint32_t r = r0 + mine, row = cut.row0 + r;
        const bool live = row < cut.rows;
        float top = -INFINITY, sum = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float m, float l, const float4& o) {
            if (m == -INFINITY && l == 0.0f) return;                      // saw nothing
            const float to = fmaxf(top, m), f0 = top == to ? 1.0f : ex2(top - to), f1 = m == to ? 1.0f : ex2(m - to);
            top = to;
            sum = sum * f0 + l * f1;
            v.x = v.x * f0 + o.x * f1; v.y = v.y * f0 + o.y * f1; v.z = v.z * f0 + o.z * f1; v.w = v.w * f0 + o.w * f1;
        };
        constexpr uint32_t U = 4;                                         // parts that a thread has under way
        for (uint32_t i0 = way; live && i0 < cut.parts; i0 += WAYS * U) {
            float2 ml[U];
            float4 o[U];
#pragma unroll
            for (uint32_t k = 0; k < U; ++k) {
                const uint32_t i = i0 + WAYS * k;
                ml[k] = make_float2(-INFINITY, 0.0f);
                if (i < cut.parts) {
                    // part 0 is this block's second, part i the first of block + i
                    const float* at = base + (size_t)(i == 0 ? 1u : 2u * i) * kv4_part_floats(D, NT);
                    ml[k] = __ldcg(reinterpret_cast<const float2*>(at + 8 * NT * D + 2 * r));
                    o[k] = __ldcg(reinterpret_cast<const float4*>(at + r * D + 4 * d4));
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < U; ++k) add(ml[k].x, ml[k].y, o[k]);
        }
        s_v[mine][way][d4] = v;
        if (d4 == 0) { s_ml[mine][way][0] = top; s_ml[mine][way][1] = sum; }
        __syncthreads();
        if (way == 0 && live) {
#pragma unroll
            for (uint32_t w = 1; w < WAYS; ++w) add(s_ml[mine][w][0], s_ml[mine][w][1], s_v[mine][w][d4]);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const long long tok = cut.start + row / p.ratio, h = cut.head * p.ratio + row % p.ratio;
            T* dst = reinterpret_cast<T*>(p.out) + tok * p.out_token + h * p.out_head + 4 * d4;
            T o[4] = {Tr<DT>::from_f(v.x * inv), Tr<DT>::from_f(v.y * inv), Tr<DT>::from_f(v.z * inv), Tr<DT>::from_f(v.w * inv)};
            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
            if (p.lse && d4 == 0) p.lse[(size_t)tok * p.kv_heads * p.ratio + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
        }
        __syncthreads();                                                  // the sums in shared memory are the next rows'
    }
}

// ---- launch, one translation unit per head size ------------------------------------------------------------
template <int D, int GS, int NT, int DT> int decode_blocks_per_sm() {
    static int per_sm[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (!per_sm[dev]) {
        const size_t smem = decode_smem<D, GS, NT>();
        int n = 0;
        if (cudaFuncSetAttribute(kv4_decode_kernel<D, GS, NT, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv4_decode_kernel<D, GS, NT, DT>, kDecodeThreads, smem) != cudaSuccess || n < 1)
            return 0;
        per_sm[dev] = n;
    }
    return per_sm[dev];
}

template <int D, int GS, int NT, int DT> cudaError_t run_decode(const Kv4Attn& p, uint32_t blocks, cudaStream_t s) {
    if (!decode_blocks_per_sm<D, GS, NT, DT>()) return cudaErrorInvalidConfiguration;
    if (cudaError_t e = launch_early(kv4_decode_kernel<D, GS, NT, DT>, dim3(blocks), dim3(kDecodeThreads), decode_smem<D, GS, NT>(), s, p)) return e;
    return launch_early(kv4_join_kernel<D, NT, DT>, dim3(blocks, 8 * NT / kJoinRows), dim3(JoinShape<D>::kThreads), 0, s, p, blocks);
}

// f<GS, NT, DT>() of a head size
template <int D, typename F> auto for_decode(uint32_t group, uint32_t nt, int dt, F&& f) -> decltype(f.template operator()<32, 1, FP16>()) {
#define KV4_CASE(G_, N_)                                                                                                             \
    if constexpr (G_ <= D && (N_ == 1 || D <= 128))                                                                                  \
        if (group == G_ && nt == N_) return dt == FP16 ? f.template operator()<G_, N_, FP16>() : f.template operator()<G_, N_, BF16>()
    KV4_CASE(32, 1);
    KV4_CASE(64, 1);
    KV4_CASE(128, 1);
    KV4_CASE(32, 2);
    KV4_CASE(64, 2);
    KV4_CASE(128, 2);
#undef KV4_CASE
    return f.none();
}

template <int D> struct BlocksCall {
    int none() { return 0; }
    template <int GS, int NT, int DT> int operator()() { return decode_blocks_per_sm<D, GS, NT, DT>(); }
};
template <int D> struct DecodeCall {
    const Kv4Attn& p;
    uint32_t blocks;
    cudaStream_t s;
    cudaError_t none() { return cudaErrorInvalidValue; }
    template <int GS, int NT, int DT> cudaError_t operator()() { return run_decode<D, GS, NT, DT>(p, blocks, s); }
};

}  // namespace dd
