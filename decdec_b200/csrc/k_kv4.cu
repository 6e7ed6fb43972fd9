// Around the 4-bit key/value cache: rotary positions, the plan of a step, new rows into the cache and rows back out of it.
#include "internal.h"
#include "kv4.cuh"
#include "../../include/decdec_b200.h"

#include <cstdio>

namespace dd {
namespace {

constexpr uint32_t kMaxRotaryPairs = 512;

// ---- rotary positions ------------------------------------------------------------------------------------
// (a, b) -> ((a cos - b sin) f, (b cos + a sin) f), angle = position * frequency.  Bound by memory: 16-bit rows are read and
// written once, V pairs (2 V elements, 16 bytes a half) per thread and step.  The angle is taken in 64 bits, where a position of a
// million still has 2^-33 of a turn, reduced to one turn there, and its sine and cosine in 32 bits: once per token and pair, in
// shared memory for all heads.  A block takes `span` tokens, so that its threads have an angle each, and reads its first rows before
// it computes them.
template <int DT, bool HALF, int V>
__global__ void __launch_bounds__(256) rotary_kernel(Rows q, uint32_t q_heads, Rows k, uint32_t k_heads, Rows qo, Rows ko, const void* positions,
                                                     int wide, const double* __restrict__ frequencies, uint32_t tokens, uint32_t head_dim,
                                                     uint32_t rotary_dim, uint32_t span, float factor) {
    using T = typename Tr<DT>::T;
    extern __shared__ float2 turn[];                          // [span][rotary_dim / 2]
    struct alignas(sizeof(T) * V) Vec { T v[V]; };
    pdl_trigger();
    pdl_wait();
    const uint32_t pairs = rotary_dim / 2u;
    const uint32_t t0 = blockIdx.x * span, n = min(span, tokens - t0);
    // steps of a head: pairs / V that turn, then (head_dim - rotary_dim) / 2V that are copied
    const uint32_t turning = pairs / V, steps = head_dim / (2u * V), per_token = (q_heads + k_heads) * steps, total = n * per_token;
    struct At { const T* src; T* dst; uint32_t at0, at1, angle; bool turns; };
    auto place = [&](uint32_t j) {
        const uint32_t t = span == 1u ? 0u : j / per_token;
        const uint32_t in = j - t * per_token;
        uint32_t h = in / steps;
        const uint32_t e = in - h * steps;
        const bool is_k = h >= q_heads;
        if (is_k) h -= q_heads;
        At a;
        a.src = reinterpret_cast<const T*>(is_k ? k.p : q.p) + (long long)(t0 + t) * (is_k ? k.token : q.token) + (long long)h * (is_k ? k.head : q.head);
        a.dst = reinterpret_cast<T*>(const_cast<void*>(is_k ? ko.p : qo.p)) + (long long)(t0 + t) * (is_k ? ko.token : qo.token) +
                (long long)h * (is_k ? ko.head : qo.head);
        a.turns = e < turning;
        // half layout: the two halves of a pair are rotary_dim / 2 apart; else, and where elements are only copied, neighbours
        a.at0 = (HALF && a.turns) ? e * V : e * 2u * V;
        a.at1 = (HALF && a.turns) ? a.at0 + pairs : a.at0 + V;
        a.angle = t * pairs + e * V;
        return a;
    };
    uint32_t j = blockIdx.y * blockDim.x + threadIdx.x;
    At at = {};
    Vec x, y;
    if (j < total) {
        at = place(j);
        x = *reinterpret_cast<const Vec*>(at.src + at.at0);
        y = *reinterpret_cast<const Vec*>(at.src + at.at1);
    }
    for (uint32_t i = threadIdx.x; i < n * pairs; i += blockDim.x) {
        const uint32_t t = t0 + i / pairs;
        const long long pos = wide ? reinterpret_cast<const long long*>(positions)[t] : (long long)reinterpret_cast<const int*>(positions)[t];
        const double turns = (double)pos * frequencies[i % pairs] * 0.15915494309189533576888;     // 1 / 2 pi
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    while (j < total) {
        if (at.turns) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                T& xa = HALF ? x.v[i] : (2 * i < V ? x.v[(2 * i) % V] : y.v[(2 * i) % V]);
                T& xb = HALF ? y.v[i] : (V == 1 ? y.v[0] : (2 * i < V ? x.v[(2 * i + 1) % V] : y.v[(2 * i + 1) % V]));
                const float2 cs = turn[at.angle + i];
                const float a = Tr<DT>::to_f(xa), b = Tr<DT>::to_f(xb);
                xa = Tr<DT>::from_f((a * cs.x - b * cs.y) * factor);
                xb = Tr<DT>::from_f((b * cs.x + a * cs.y) * factor);
            }
        }
        *reinterpret_cast<Vec*>(at.dst + at.at0) = x;
        *reinterpret_cast<Vec*>(at.dst + at.at1) = y;
        j += blockDim.x * gridDim.y;
        if (j < total) {
            at = place(j);
            x = *reinterpret_cast<const Vec*>(at.src + at.at0);
            y = *reinterpret_cast<const Vec*>(at.src + at.at1);
        }
    }
}

template <int DT, bool HALF>
cudaError_t rotary_any(int vec, dim3 grid, uint32_t span, cudaStream_t s, const Rows& q, uint32_t qh, const Rows& k, uint32_t kh, const Rows& qo, const Rows& ko,
                       const void* positions, int wide, const double* f, uint32_t tokens, uint32_t d, uint32_t r, float factor) {
    constexpr int W = DT == FP32 ? 4 : 8;
    return launch_early(vec ? rotary_kernel<DT, HALF, W> : rotary_kernel<DT, HALF, 1>, grid, dim3(256), (size_t)span * r / 2u * sizeof(float2), s, q, qh, k, kh, qo, ko,
                        positions, wide, f, tokens, d, r, span, factor);
}

// ---- plan of a step --------------------------------------------------------------------------------------
// One launch, no pass over the requests that another waits for: every thread block sums all requests' tokens and new pages itself
// (a few kilobytes), then takes its share of the tokens and finds each token's request by bisection.  A block's threads hold
// consecutive runs of requests; `at` are the sums before each run.
constexpr int kPlanThreads = 512;

struct Plan {
    const int32_t *lengths, *fresh;
    int32_t* table;
    long long table_stride;
    const int32_t *free_pages, *free_count;
    long long *positions, *slots;
    int32_t *starts, *out_lengths, *out_free, *status;
    uint32_t requests, table_cols, free_cap, page, tokens;
};

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    return v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(Plan p) {
    __shared__ long long at_tok[kPlanThreads + 1], at_page[kPlanThreads + 1];
    __shared__ long long warp_tok[kPlanThreads / 32], warp_page[kPlanThreads / 32];
    pdl_trigger();
    pdl_wait();
    const uint32_t run = (p.requests + kPlanThreads - 1u) / kPlanThreads;
    const uint32_t b0 = min(threadIdx.x * run, p.requests), b1 = min(b0 + run, p.requests);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long cap = (long long)p.table_cols * p.page;
    long long tok = 0, pages = 0;
    int bad = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        const long long have = p.lengths[b], n = p.fresh[b];
        if (have < 0 || n < 0) { bad |= 8; continue; }
        if (have + n > cap) bad |= 2;
        tok += n;
        pages += (have + n + p.page - 1) / p.page - (have + p.page - 1) / p.page;
    }
    const long long tok_in = warp_scan(tok, lane), pages_in = warp_scan(pages, lane);
    if (lane == 31) { warp_tok[warp] = tok_in; warp_page[warp] = pages_in; }
    bad = __reduce_or_sync(0xffffffffu, bad);
    const int any2 = __syncthreads_or(bad & 2), any8 = __syncthreads_or(bad & 8);
    long long before_tok = 0, before_page = 0, all_tok = 0, all_page = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) { before_tok += warp_tok[w]; before_page += warp_page[w]; }
        all_tok += warp_tok[w];
        all_page += warp_page[w];
    }
    at_tok[threadIdx.x] = before_tok + tok_in - tok;
    at_page[threadIdx.x] = before_page + pages_in - pages;
    if (threadIdx.x == 0) { at_tok[kPlanThreads] = all_tok; at_page[kPlanThreads] = all_page; }
    __syncthreads();
    const long long count = p.free_count[0];
    int status = (any2 ? 2 : 0) | (any8 ? 8 : 0);
    if (all_page > count || count > (long long)p.free_cap || count < 0) status |= 1;
    if (all_tok > (long long)p.tokens) status |= 4;
    if (blockIdx.x == 0) {
        long long s = at_tok[threadIdx.x];
        for (uint32_t b = b0; b < b1; ++b) {
            const int32_t have = p.lengths[b], n = p.fresh[b];
            p.starts[b] = status ? 0 : (int32_t)s;
            p.out_lengths[b] = status ? have : have + n;
            s += n;
        }
        if (threadIdx.x == 0) {
            p.starts[p.requests] = status ? 0 : (int32_t)all_tok;
            p.out_free[0] = (int32_t)(status ? count : count - all_page);
            p.status[0] = status;
        }
    }
    for (uint32_t t = blockIdx.x * kPlanThreads + threadIdx.x; t < p.tokens; t += gridDim.x * kPlanThreads) {
        long long pos = 0, slot = -1;
        if (!status && (long long)t < all_tok) {
            int lo = 0, hi = kPlanThreads;                     // the last run that begins at or before t and is not empty
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (at_tok[mid] <= (long long)t) lo = mid; else hi = mid;
            }
            long long s = at_tok[lo], pg = at_page[lo];
            uint32_t b = (uint32_t)lo * run;
            int32_t have = p.lengths[b], n = p.fresh[b];
            while ((long long)t >= s + n) {                    // ends inside the run: t lies below the next run's sum
                s += n;
                pg += ((long long)have + n + p.page - 1) / p.page - ((long long)have + p.page - 1) / p.page;
                ++b;
                have = p.lengths[b];
                n = p.fresh[b];
            }
            pos = have + ((long long)t - s);
            const uint32_t column = (uint32_t)pos / p.page, used = ((uint32_t)have + p.page - 1u) / p.page;
            int32_t page;
            if (column >= used) {
                page = p.free_pages[count - 1 - (pg + (column - used))];
                // its first token enters a new page into the table, which nobody reads at that place
                if ((uint32_t)pos % p.page == 0u) p.table[(long long)b * p.table_stride + column] = page;
            } else {
                page = p.table[(long long)b * p.table_stride + column];
            }
            slot = (long long)page * p.page + (uint32_t)pos % p.page;
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
}

// ---- rows into the cache -----------------------------------------------------------------------------------
// a register of two 16-bit values
template <int DT> struct Two;
template <> struct Two<FP16> { using T = __half2; };
template <> struct Two<BF16> { using T = __nv_bfloat162; };
template <int DT> __device__ __forceinline__ typename Two<DT>::T as2(uint32_t v) { return *reinterpret_cast<const typename Two<DT>::T*>(&v); }
template <int DT> __device__ __forceinline__ uint32_t bits2(typename Two<DT>::T v) { return *reinterpret_cast<const uint32_t*>(&v); }
// the smaller of each, NaN if one is
template <int DT> __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) { return bits2<DT>(__hmin2_nan(as2<DT>(a), as2<DT>(b))); }
// whether one of the two 16-bit values is infinite or NaN
template <int DT> __device__ __forceinline__ uint32_t no_number(uint32_t v) {
    constexpr uint32_t E = DT == FP16 ? 0x7c007c00u : 0x7f807f80u, U = DT == FP16 ? 0x04000400u : 0x00800080u;
    return ((v & E) + U) & 0x80008000u;
}

// code of x in steps from lo, the nearest, ties to even, exactly as over the reals: the two comparisons of the guess n with its borders in
// exact arithmetic (difference with its rounding error; border * step has 16 bits).  All arguments halved, so that the range of a bf16
// group does not overflow.
__device__ __forceinline__ float exact_code(float xh, float loh, float steph, float n) {
    const float d = xh - loh;
    const float back = d + loh;                                  // two-difference: xh - loh = d + e
    const float e = (xh - back) + ((back - d) - loh);
    n = fminf(fmaxf(n, 0.0f), 15.0f);
    const bool odd = ((int)n & 1) != 0;
    const float above = fmaf(-(n + 0.5f), steph, d) + e, below = fmaf(-(n - 0.5f), steph, d) + e;
    if (above > 0.0f || (above == 0.0f && odd)) n += 1.0f;
    else if (below < 0.0f || (below == 0.0f && odd)) n -= 1.0f;
    return fminf(fmaxf(n, 0.0f), 15.0f);
}

// (hi - lo) / 15 rounded to the type as over the reals, of halves.  The quotient by a constant is corrected by its remainder, which rounds as
// a division does (Markstein's theorem) where nothing underflows: it is off by less than two units of 32 bits.  That is too much only next to
// the middle of two numbers of the type.  15 times a middle is an odd multiple of a 2^12th (fp16; bf16: 2^9th) of the step's power of two, so the
// range comes that near without meeting it only by a small end of the group whose own last bit lies 2^-25 below the range: fp16 alone has such
// (bf16: 2^-19), and no subnormal steps, whose ranges are whole multiples of 2^-24.  There the range is compared with 15 middles exactly.
template <int DT> __device__ __forceinline__ float step_of(float lo, float hi) {
    const float a = 0.5f * hi, b = 0.5f * lo, range = a - b;
    float q = range * (1.0f / 7.5f);
    q = fmaf(fmaf(-q, 7.5f, range), 1.0f / 7.5f, q);
    if (range < 1e-30f) q = range / 7.5f;
    if constexpr (DT == FP16) {
        const uint32_t bits = __float_as_uint(q);
        if ((bits & 0x1fffu) - 0xffcu <= 8u) {                       // of the 13 bits that fp16 leaves off; about one group in 2^10
            const uint32_t middle = (bits & ~0x1fffu) | 0x1000u;
            const float back = range + b, e = (a - back) + ((back - range) - b);      // a - b = range + e
            const float over = fmaf(-7.5f, __uint_as_float(middle), range) + e;
            q = __uint_as_float(middle + (over > 0.0f) - (over < 0.0f));
        }
    }
    return Tr<DT>::to_f(Tr<DT>::from_f(q));
}

// eight codes of 16-bit values in a word
template <int DT> __device__ __forceinline__ uint32_t code_word(const uint4& x, float lo, float step) {
    if (!(step > 0.0f)) return 0u;
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
    const float loh = 0.5f * lo, steph = 0.5f * step;
    const bool small = steph < 1e-30f;                           // its reciprocal may overflow
    float inv;                                                   // a guess: what it is off by stays far below `near`
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(steph));
    if (small) inv = 0.0f;
    const float near = steph * 0.4999f;
    // a normal step is off by 2^-8 at most, so no quotient comes near 15.5; a subnormal one may be off by half of it
    bool border = step < (DT == FP16 ? 6.103515625e-5f : 1.17549435e-38f) || small;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float four = 0.0f;                                       // the codes as digits, which 24 bits hold
#pragma unroll
        for (int k = 3; k >= 0; --k) {
            const float2 f = unpack2<DT>(u[2 * i + k / 2]);
            const float d = fmaf(0.5f, k & 1 ? f.y : f.x, -loh); // the product is exact
            const float n = fmaf(d, inv, 12582912.0f) - 12582912.0f;         // 1.5 * 2^23: the sum is rounded to a whole number
            border |= fabsf(fmaf(-n, steph, d)) > near;          // next to a border
            four = fmaf(four, 16.0f, n);
        }
        word |= (__float_as_uint(four + 8388608.0f) & 0xffffu) << (16 * i);
    }
    if (border) {                                                // of the eight, about one in 2^9 random ones; more in short types
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = unpack2<DT>(u[i / 2]);
            const float h = 0.5f * (i & 1 ? f.y : f.x), d = h - loh;
            word |= (uint32_t)exact_code(h, loh, steph, small ? rintf(d / steph) : rintf(d * inv)) << (4 * i);
        }
    }
    return word;
}

// where a slot lies: the first head's cell and the token's place in it
struct Place {
    uint8_t* cell;
    uint32_t r;
    bool inside;
};
__device__ __forceinline__ Place place_of(const Kv4Cache& c, const void* slots, int wide, uint32_t t, uint32_t cell_bytes, bool report, unsigned* err) {
    const long long slot = wide ? reinterpret_cast<const long long*>(slots)[t] : (long long)reinterpret_cast<const int*>(slots)[t];
    const uint32_t page_tokens = c.page_cells * kCellTokens;
    Place p;
    p.inside = slot >= 0 && slot < (long long)c.pages * page_tokens;
    if (slot >= 0 && !p.inside && report) raise_error(err, kErrKv4Page);
    const uint32_t page = p.inside ? quotient((size_t)slot, page_tokens) : 0u;
    const uint32_t in_page = p.inside ? (uint32_t)((size_t)slot - (size_t)page * page_tokens) : 0u;
    p.cell = c.data + (size_t)page * c.kv_heads * c.page_bytes + (size_t)(in_page / kCellTokens) * cell_bytes;
    p.r = in_page % kCellTokens;
    return p;
}

// How a warp lies on a token: eight elements a lane, so 8 or 16 lanes on a head (128 of its elements if there are 256), the keys of all
// heads of a round on the first half of the warp and their values on the second.
template <int D> struct Lanes {
    static constexpr uint32_t kBlock = D < 128 ? D : 128;           // elements of a unit
    static constexpr uint32_t kUnit = kBlock / 8;                   // lanes of a unit
    static constexpr uint32_t kUnits = D / kBlock;                  // units of a head
    static constexpr uint32_t kRound = 16 / kUnit;                  // units of a round, keys and values
};

constexpr uint32_t kRounds = 4;                                     // of a warp at most

// A warp takes a token and `rounds` rounds of its heads, which are coalesced 256-byte reads of keys and values; the group extremes are a
// few shuffles of (least, -largest) pairs.  Bound by waiting: two dependent round trips (slot, row), and value codes that lie in pieces of two
// bytes, four to every 16 bytes and those 64 bytes apart.  Issue slots are 49 % busy (224 instructions for the keys and values of a head of 128),
// memory 15 %.  8191 tokens of 10 heads of 128, written and read back: the slot for every head, divisions and float extremes 84 us, the slot once
// and packed extremes 51, approximate reciprocals and an exact correction 47 to 49, steps rounded exactly 50; eight elements a lane, and all reads
// at once, the same.
template <int DT, int D, int GS, bool VEC>
__global__ void __launch_bounds__(256) append_kernel(Rows k, Rows v, const void* slots, int wide, Kv4Cache c, uint32_t tokens, uint32_t chunks, uint32_t rounds,
                                                     unsigned* err) {
    using T = typename Tr<DT>::T;
    using L = Lanes<D>;
    constexpr int GL = GS / 8;                           // lanes of a group
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, all = c.kv_heads * L::kUnits;
    const bool side = lane >= 16u;
    const Rows& x = side ? v : k;
    const uint64_t items = (uint64_t)tokens * chunks;
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x / 32u) + (threadIdx.x >> 5); i < items; i += (uint64_t)gridDim.x * (blockDim.x / 32u)) {
        const uint32_t t = quotient(i, chunks), chunk = (uint32_t)(i - (uint64_t)t * chunks);
        const Place at = place_of(c, slots, wide, t, kv4_cell_bytes(D, GS), lane == 0u && chunk == 0u, err);
        if (!at.inside) continue;
        const T* row = reinterpret_cast<const T*>(x.p) + (long long)t * x.token;
        const uint32_t first = chunk * rounds * L::kRound + (lane & 15u) / L::kUnit;
        uint4 all_raw[kRounds];
#pragma unroll
        for (uint32_t round = 0; round < kRounds; ++round) {         // everything that the warp reads is under way at once
            const uint32_t unit = first + round * L::kRound;
            all_raw[round] = make_uint4(0, 0, 0, 0);
            if (round < rounds && unit < all) {
                const T* src = row + (long long)(unit / L::kUnits) * x.head + unit % L::kUnits * L::kBlock + lane % L::kUnit * 8u;
                if constexpr (VEC) {
                    all_raw[round] = *reinterpret_cast<const uint4*>(src);
                } else {
                    const uint16_t* w = reinterpret_cast<const uint16_t*>(src);
                    all_raw[round] = make_uint4((uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16,
                                                (uint32_t)w[4] | (uint32_t)w[5] << 16, (uint32_t)w[6] | (uint32_t)w[7] << 16);
                }
            }
        }
#pragma unroll
        for (uint32_t round = 0; round < kRounds; ++round) {
            if (round >= rounds) break;
            const uint32_t unit = first + round * L::kRound;
            const bool live = unit < all;
            const uint32_t h = live ? unit / L::kUnits : 0u, e = unit % L::kUnits * L::kBlock + lane % L::kUnit * 8u;
            const uint4 raw = all_raw[round];
            // (least, -largest): a minimum over both signs, then over the lanes of the group.  One that is no number comes through, and the
            // group reads back as NaN
            const uint32_t s = 0x80008000u;
            const uint32_t low = min2<DT>(min2<DT>(raw.x, raw.y), min2<DT>(raw.z, raw.w));
            const uint32_t high = min2<DT>(min2<DT>(raw.x ^ s, raw.y ^ s), min2<DT>(raw.z ^ s, raw.w ^ s));
            uint32_t range = min2<DT>(__byte_perm(low, high, 0x5410), __byte_perm(low, high, 0x7632));
#pragma unroll
            for (int o = 1; o < GL; o *= 2) range = min2<DT>(range, __shfl_xor_sync(0xffffffffu, range, o));
            const float2 lh = unpack2<DT>(range);
            float lo = lh.x, step = step_of<DT>(lo, -lh.y);
            if (no_number<DT>(range)) { lo = __int_as_float(0x7fc00000); step = 0.0f; }
            const uint32_t word = code_word<DT>(raw, lo, step);
            if (live) {
                uint8_t* cell = at.cell + (size_t)h * c.page_bytes;
                if (!side) {
                    *reinterpret_cast<uint32_t*>(cell + kv4_key_word(D, at.r, e / 4u)) = word;       // its halves are neighbours
                } else {
                    *reinterpret_cast<uint16_t*>(cell + kv4_value_word(D, at.r, e / 4u)) = (uint16_t)word;
                    *reinterpret_cast<uint16_t*>(cell + kv4_value_word(D, at.r, e / 4u + 1u)) = (uint16_t)(word >> 16);
                }
                if (e % GS == 0u)
                    *reinterpret_cast<uint32_t*>(cell + (side ? kv4_value_step(D, GS, at.r, e / GS) : kv4_key_step(D, GS, at.r, e / GS))) = pack2<DT>(step, lo);
            }
        }
    }
}

// ---- rows out of the cache -----------------------------------------------------------------------------------
// Bound by waiting, as append is: issue slots 38 % busy, memory 6 %.  Warps and lanes as in append.
template <int DT, int D, int GS>
__global__ void __launch_bounds__(256) gather_kernel(Kv4Cache c, const void* slots, int wide, void* k_out, void* v_out, uint32_t tokens, uint32_t chunks,
                                                     uint32_t rounds, unsigned* err) {
    using T = typename Tr<DT>::T;
    using L = Lanes<D>;
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, all = c.kv_heads * L::kUnits;
    const bool side = lane >= 16u;
    const uint64_t items = (uint64_t)tokens * chunks;
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x / 32u) + (threadIdx.x >> 5); i < items; i += (uint64_t)gridDim.x * (blockDim.x / 32u)) {
        const uint32_t t = quotient(i, chunks), chunk = (uint32_t)(i - (uint64_t)t * chunks);
        const Place at = place_of(c, slots, wide, t, kv4_cell_bytes(D, GS), lane == 0u && chunk == 0u, err);
        const uint32_t first = chunk * rounds * L::kRound + (lane & 15u) / L::kUnit;
        T* row = reinterpret_cast<T*>(side ? v_out : k_out) + (size_t)t * c.kv_heads * D;
        uint32_t all_w[kRounds], all_s[kRounds];
#pragma unroll
        for (uint32_t round = 0; round < kRounds; ++round) {         // everything that the warp reads is under way at once
            const uint32_t unit = first + round * L::kRound, h = unit / L::kUnits, e = unit % L::kUnits * L::kBlock + lane % L::kUnit * 8u;
            all_w[round] = all_s[round] = 0u;
            if (at.inside && round < rounds && unit < all) {
                const uint8_t* cell = at.cell + (size_t)h * c.page_bytes;
                all_w[round] = side ? (uint32_t)*reinterpret_cast<const uint16_t*>(cell + kv4_value_word(D, at.r, e / 4u)) |
                                          (uint32_t)*reinterpret_cast<const uint16_t*>(cell + kv4_value_word(D, at.r, e / 4u + 1u)) << 16
                                    : *reinterpret_cast<const uint32_t*>(cell + kv4_key_word(D, at.r, e / 4u));
                all_s[round] = *reinterpret_cast<const uint32_t*>(cell + (side ? kv4_value_step(D, GS, at.r, e / GS) : kv4_key_step(D, GS, at.r, e / GS)));
            }
        }
#pragma unroll
        for (uint32_t round = 0; round < kRounds; ++round) {
            if (round >= rounds) break;
            const uint32_t unit = first + round * L::kRound, h = unit / L::kUnits, e = unit % L::kUnits * L::kBlock + lane % L::kUnit * 8u;
            const uint32_t w = all_w[round], s = all_s[round];
            // offset + step * code in one rounding, kept finite (a rounded step may lead beyond the type): pairs (0, 4), (1, 5), (2, 6), (3, 7)
            constexpr uint32_t BASE = DT == FP16 ? 0x64006400u : 0x43004300u, MOST = DT == FP16 ? 0x7bff7bffu : 0x7f7f7f7fu;      // 1024 or 128
            const auto step2 = as2<DT>(__byte_perm(s, 0, 0x1010)), lo2 = as2<DT>(__byte_perm(s, 0, 0x3232));
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j] = min2<DT>(bits2<DT>(__hfma2(__hsub2(as2<DT>((w >> (4 * j) & 0x000f000fu) | BASE), as2<DT>(BASE)), step2, lo2)), MOST);
            if (unit < all)
                *reinterpret_cast<uint4*>(row + (size_t)h * D + e) = make_uint4(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410),
                                                                               __byte_perm(o[0], o[1], 0x7632), __byte_perm(o[2], o[3], 0x7632));
        }
    }
}

// how a token's heads are cut: up to four rounds to a warp while there are tokens enough to fill the device, else fewer
struct Cut {
    uint32_t chunks, rounds, blocks;
};
Cut cut_heads(uint32_t tokens, uint32_t kv_heads, uint32_t d) {
    const uint32_t widths = (kv_heads * d + 127u) / 128u;                  // rounds of a token
    const uint32_t want = device_sms() * 32u;                              // warps
    Cut c;
    c.chunks = tokens >= want ? 1u : (want + tokens - 1u) / tokens;
    if (c.chunks < (widths + kRounds - 1u) / kRounds) c.chunks = (widths + kRounds - 1u) / kRounds;
    if (c.chunks > widths) c.chunks = widths;
    c.rounds = (widths + c.chunks - 1u) / c.chunks;
    c.chunks = (widths + c.rounds - 1u) / c.rounds;
    const uint64_t blocks = ((uint64_t)tokens * c.chunks + 7u) / 8u;
    c.blocks = (uint32_t)(blocks < 0x40000000ull ? blocks : 0x40000000ull);
    return c;
}

template <int DT, int D, int GS>
cudaError_t run_append(const Rows& k, const Rows& v, const void* slots, int wide, const Kv4Cache& c, uint32_t tokens, bool vec, unsigned* err, cudaStream_t s) {
    const Cut cut = cut_heads(tokens, c.kv_heads, D);
    return launch_early(vec ? append_kernel<DT, D, GS, true> : append_kernel<DT, D, GS, false>, dim3(cut.blocks), dim3(256), 0, s, k, v, slots, wide, c, tokens,
                        cut.chunks, cut.rounds, err);
}

template <int DT, int D, int GS>
cudaError_t run_gather(const Kv4Cache& c, const void* slots, int wide, void* k, void* v, uint32_t tokens, unsigned* err, cudaStream_t s) {
    const Cut cut = cut_heads(tokens, c.kv_heads, D);
    return launch_early(gather_kernel<DT, D, GS>, dim3(cut.blocks), dim3(256), 0, s, c, slots, wide, k, v, tokens, cut.chunks, cut.rounds, err);
}

// f.template operator()<DT, D, GS>() for the types, heads and groups that the cache takes
template <typename F> cudaError_t for_format(int dt, uint32_t d, uint32_t group, F&& f) {
#define KV4_CASE(D_, G_) \
    if (d == D_ && group == G_) return dt == FP16 ? f.template operator()<FP16, D_, G_>() : f.template operator()<BF16, D_, G_>()
    KV4_CASE(64, 32);
    KV4_CASE(64, 64);
    KV4_CASE(128, 32);
    KV4_CASE(128, 64);
    KV4_CASE(128, 128);
    KV4_CASE(256, 32);
    KV4_CASE(256, 64);
    KV4_CASE(256, 128);
#undef KV4_CASE
    return cudaErrorInvalidValue;
}

struct AppendCall {
    const Rows &k, &v;
    const void* slots;
    int wide;
    const Kv4Cache& c;
    uint32_t tokens;
    bool vec;
    unsigned* err;
    cudaStream_t s;
    template <int DT, int D, int GS> cudaError_t operator()() { return run_append<DT, D, GS>(k, v, slots, wide, c, tokens, vec, err, s); }
};

struct GatherCall {
    const Kv4Cache& c;
    const void* slots;
    int wide;
    void *k, *v;
    uint32_t tokens;
    unsigned* err;
    cudaStream_t s;
    template <int DT, int D, int GS> cudaError_t operator()() { return run_gather<DT, D, GS>(c, slots, wide, k, v, tokens, err, s); }
};

int fail(int code, const char* fmt, unsigned long long a = 0, unsigned long long b = 0) {
    char msg[256];
    snprintf(msg, sizeof(msg), fmt, a, b);
    return set_last_error(code, msg);
}

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return 0;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s failed: %s", what, cudaGetErrorString(e));
    return set_last_error(DECDEC_E_CUDA, msg);
}

int check_format(int dtype, uint32_t head_dim, uint32_t group, uint32_t page, const void* cache, uint32_t pages, uint32_t kv_heads) {
    if (dtype != FP16 && dtype != BF16) return fail(DECDEC_E_INVALID, "the 4-bit cache supports half and bfloat16 only.");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(DECDEC_E_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %llu", head_dim);
    if ((group != 32 && group != 64 && group != 128) || group > head_dim)
        return fail(DECDEC_E_INVALID, "group_size must be 32, 64 or 128 and not above head_dim, got %llu", group);
    if (page == 0 || page % kCellTokens || page > 65536u) return fail(DECDEC_E_INVALID, "page_size must be a multiple of 16 up to 65536, got %llu", page);
    if (!cache || (reinterpret_cast<uintptr_t>(cache) & 15u)) return fail(DECDEC_E_INVALID, "the cache must be 16-byte aligned device memory");
    if (pages == 0 || kv_heads == 0) return fail(DECDEC_E_INVALID, "empty cache");
    if (pages > 0x7fffffffu) return fail(DECDEC_E_INVALID, "too many pages");
    return 0;
}

Kv4Cache make_cache(const void* cache, uint32_t pages, uint32_t page, uint32_t kv_heads, uint32_t d, uint32_t group) {
    Kv4Cache c;
    c.data = reinterpret_cast<uint8_t*>(const_cast<void*>(cache));
    c.pages = pages; c.page_cells = page / kCellTokens; c.kv_heads = kv_heads; c.head_dim = d; c.group = group;
    c.page_bytes = c.page_cells * kv4_cell_bytes(d, group);
    return c;
}

// whether vectors of `elems` elements of `size` bytes may be read at every row
bool aligned(const void* p, long long token, long long head, long long elems, int size) {
    return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)(elems * size)) == 0 && token % elems == 0 && head % elems == 0;
}

}  // namespace

cudaError_t launch_rotary(int dt, const Rows& q, uint32_t q_heads, const Rows& k, uint32_t k_heads, void* q_out, long long qo_token,
                          long long qo_head, void* k_out, long long ko_token, long long ko_head, const void* positions, int wide,
                          const double* f, uint32_t tokens, uint32_t d, uint32_t r, int interleaved, float factor, cudaStream_t s) {
    const int size = dt == FP32 ? 4 : 2, W = dt == FP32 ? 4 : 8;
    const Rows qo{q_out, qo_token, qo_head}, ko{k_out, ko_token, ko_head};
    int vec = (r / 2u) % W == 0 && (d - r) % (2 * W) == 0;
    for (const Rows* x : {&q, &k, &qo, &ko})
        if (x->p) vec &= aligned(x->p, x->token, x->head, W, size);
    // several tokens to a block while there are blocks enough for every SM (8192 tokens of 40 heads of 128: 34 us, one to a block 38); where
    // there are few tokens, they are cut by heads
    const uint32_t steps = (q_heads + k_heads) * d / (2u * (vec ? W : 1));
    uint32_t span = 1, cut = 1;
    while (span < 4u && tokens / (2u * span) >= 8u * device_sms() && 2u * span * r / 2u <= 2u * kMaxRotaryPairs) span *= 2u;
    if (span == 1u) {
        cut = (2u * device_sms() + tokens - 1u) / tokens;
        const uint32_t most = (steps + 255u) / 256u;
        if (cut > most) cut = most;
        if (cut == 0) cut = 1;
    }
    const dim3 grid((tokens + span - 1u) / span, cut);
#define ROTARY(DT_) return interleaved ? rotary_any<DT_, false>(vec, grid, span, s, q, q_heads, k, k_heads, qo, ko, positions, wide, f, tokens, d, r, factor) \
                                       : rotary_any<DT_, true>(vec, grid, span, s, q, q_heads, k, k_heads, qo, ko, positions, wide, f, tokens, d, r, factor)
    if (dt == FP32) ROTARY(FP32);
    if (dt == FP16) ROTARY(FP16);
    ROTARY(BF16);
#undef ROTARY
}

}  // namespace dd

using namespace dd;

extern "C" {

int decdec_rotary(const void* q, int64_t q_token, int64_t q_head, uint32_t q_heads, const void* k, int64_t k_token, int64_t k_head, uint32_t k_heads,
                  void* q_out, int64_t qo_token, int64_t qo_head, void* k_out, int64_t ko_token, int64_t ko_head, const void* positions,
                  int positions_wide, const double* frequencies, uint32_t tokens, uint32_t head_dim, uint32_t rotary_dim, int interleaved,
                  float factor, int dtype, void* stream) {
    if (dtype != FP32 && dtype != FP16 && dtype != BF16) return fail(DECDEC_E_INVALID, "Unsupported data type.");
    if (head_dim == 0 || head_dim % 2u || rotary_dim % 2u || rotary_dim > head_dim || rotary_dim == 0)
        return fail(DECDEC_E_INVALID, "rotary_dim must be even, above 0 and not above head_dim (%llu of %llu)", rotary_dim, head_dim);
    if (rotary_dim > 2u * kMaxRotaryPairs) return fail(DECDEC_E_UNSUPPORTED, "rotary_dim above %llu", 2u * kMaxRotaryPairs);
    if (tokens == 0 || q_heads + k_heads == 0) return 0;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !positions || !frequencies) return fail(DECDEC_E_INVALID, "null pointer argument");
    if (tokens > 0x7fffffffu || (uint64_t)(q_heads + k_heads) * head_dim > 0x7fffffffull) return fail(DECDEC_E_UNSUPPORTED, "too many rows");
    const Rows rq{q_heads ? q : nullptr, q_token, q_head}, rk{k_heads ? k : nullptr, k_token, k_head};
    return launched(launch_rotary(dtype, rq, q_heads, rk, k_heads, q_heads ? q_out : nullptr, qo_token, qo_head, k_heads ? k_out : nullptr, ko_token, ko_head,
                                  positions, positions_wide, frequencies, tokens, head_dim, rotary_dim, interleaved, factor,
                                  reinterpret_cast<cudaStream_t>(stream)), "rotary launch");
}

int decdec_kv4_plan(const int32_t* lengths, const int32_t* fresh, uint32_t requests, int32_t* table, int64_t table_stride, uint32_t table_cols,
                    const int32_t* free_pages, uint32_t free_capacity, const int32_t* free_count, uint32_t page_size, uint32_t tokens,
                    int64_t* positions, int64_t* slots, int32_t* query_starts, int32_t* out_lengths, int32_t* out_free_count, int32_t* status,
                    void* stream) {
    if (page_size == 0 || page_size % kCellTokens || page_size > 65536u) return fail(DECDEC_E_INVALID, "page_size must be a multiple of 16 up to 65536, got %llu", page_size);
    if (!query_starts || !out_free_count || !status || !free_count || (requests && (!lengths || !fresh || !out_lengths)) || (requests && table_cols && !table) ||
        (free_capacity && !free_pages) || (tokens && (!positions || !slots)))
        return fail(DECDEC_E_INVALID, "null pointer argument");
    if (requests > 0x7fffffffu || tokens > 0x7fffffffu || table_cols > 0x7fffffffu || (uint64_t)table_cols * page_size > 0x7fffffffull)
        return fail(DECDEC_E_INVALID, "requests, tokens and the tokens of a table row must stay below 2^31");
    Plan p{lengths, fresh, table, table_stride, free_pages, free_count, reinterpret_cast<long long*>(positions), reinterpret_cast<long long*>(slots),
           query_starts, out_lengths, out_free_count, status, requests, table_cols, free_capacity, page_size, tokens};
    uint32_t blocks = (tokens + kPlanThreads - 1u) / kPlanThreads;
    if (blocks == 0) blocks = 1;
    if (blocks > device_sms()) blocks = device_sms();
    return launched(launch_early(plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, reinterpret_cast<cudaStream_t>(stream), p), "plan launch");
}

int decdec_kv4_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* slots, int slots_wide,
                      uint32_t tokens, void* cache, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                      int dtype, void* stream) {
    if (int r = check_format(dtype, head_dim, group_size, page_size, cache, pages, kv_heads)) return r;
    if (tokens == 0) return 0;
    if (!k || !v || !slots) return fail(DECDEC_E_INVALID, "null pointer argument");
    if ((uint64_t)tokens * kv_heads > 0x7fffffffull) return fail(DECDEC_E_UNSUPPORTED, "too many rows");
    unsigned* err = nullptr;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (int r = stream_error_word(s, &err)) return r;
    const Kv4Cache c = make_cache(cache, pages, page_size, kv_heads, head_dim, group_size);
    const Rows rk{k, k_token, k_head}, rv{v, v_token, v_head};
    const bool vec = aligned(k, k_token, k_head, 8, 2) && aligned(v, v_token, v_head, 8, 2);
    return launched(for_format(dtype, head_dim, group_size, AppendCall{rk, rv, slots, slots_wide, c, tokens, vec, err, s}), "append launch");
}

int decdec_kv4_gather(const void* cache, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                      const void* slots, int slots_wide, uint32_t tokens, void* k_out, void* v_out, int dtype, void* stream) {
    if (int r = check_format(dtype, head_dim, group_size, page_size, cache, pages, kv_heads)) return r;
    if (tokens == 0) return 0;
    if (!k_out || !v_out || !slots) return fail(DECDEC_E_INVALID, "null pointer argument");
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u) return fail(DECDEC_E_INVALID, "outputs must be 16-byte aligned");
    if ((uint64_t)tokens * kv_heads > 0x7fffffffull) return fail(DECDEC_E_UNSUPPORTED, "too many rows");
    unsigned* err = nullptr;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (int r = stream_error_word(s, &err)) return r;
    const Kv4Cache c = make_cache(cache, pages, page_size, kv_heads, head_dim, group_size);
    return launched(for_format(dtype, head_dim, group_size, GatherCall{c, slots, slots_wide, k_out, v_out, tokens, err, s}), "gather launch");
}

}  // extern "C"
