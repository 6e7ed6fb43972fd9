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
// shared memory for all heads.
template <int DT, bool HALF, int V>
__global__ void __launch_bounds__(256) rotary_kernel(Rows q, uint32_t q_heads, Rows k, uint32_t k_heads, Rows qo, Rows ko, const void* positions,
                                                     int wide, const double* __restrict__ frequencies, uint32_t tokens, uint32_t head_dim,
                                                     uint32_t rotary_dim, float factor) {
    using T = typename Tr<DT>::T;
    __shared__ float2 turn[kMaxRotaryPairs];
    struct alignas(sizeof(T) * V) Vec { T v[V]; };
    pdl_trigger();
    pdl_wait();
    const uint32_t pairs = rotary_dim / 2u;
    const uint32_t t = blockIdx.x;
    const long long pos = wide ? reinterpret_cast<const long long*>(positions)[t] : (long long)reinterpret_cast<const int*>(positions)[t];
    for (uint32_t i = threadIdx.x; i < pairs; i += blockDim.x) {
        const double turns = (double)pos * frequencies[i] * 0.15915494309189533576888;     // 1 / 2 pi
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    // steps of a head: pairs / V that turn, then (head_dim - rotary_dim) / 2V that are copied
    const uint32_t turning = pairs / V, steps = head_dim / (2u * V);
    const uint32_t total = (q_heads + k_heads) * steps;
    for (uint32_t j = blockIdx.y * blockDim.x + threadIdx.x; j < total; j += blockDim.x * gridDim.y) {
        uint32_t h = j / steps;
        const uint32_t e = j % steps;
        const bool is_k = h >= q_heads;
        if (is_k) h -= q_heads;
        const T* src = reinterpret_cast<const T*>(is_k ? k.p : q.p) + (long long)t * (is_k ? k.token : q.token) + (long long)h * (is_k ? k.head : q.head);
        T* dst = reinterpret_cast<T*>(const_cast<void*>(is_k ? ko.p : qo.p)) + (long long)t * (is_k ? ko.token : qo.token) +
                 (long long)h * (is_k ? ko.head : qo.head);
        const bool turns = e < turning;
        // half layout: the two halves of a pair are rotary_dim / 2 apart; else, and where elements are only copied, neighbours
        const uint32_t at0 = (HALF && turns) ? e * V : e * 2u * V;
        const uint32_t at1 = (HALF && turns) ? at0 + pairs : at0 + V;
        Vec x = *reinterpret_cast<const Vec*>(src + at0), y = *reinterpret_cast<const Vec*>(src + at1);
        if (turns) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                T& xa = HALF ? x.v[i] : (2 * i < V ? x.v[(2 * i) % V] : y.v[(2 * i) % V]);
                T& xb = HALF ? y.v[i] : (V == 1 ? y.v[0] : (2 * i < V ? x.v[(2 * i + 1) % V] : y.v[(2 * i + 1) % V]));
                const float2 cs = turn[e * V + i];
                const float a = Tr<DT>::to_f(xa), b = Tr<DT>::to_f(xb);
                xa = Tr<DT>::from_f((a * cs.x - b * cs.y) * factor);
                xb = Tr<DT>::from_f((b * cs.x + a * cs.y) * factor);
            }
        }
        *reinterpret_cast<Vec*>(dst + at0) = x;
        *reinterpret_cast<Vec*>(dst + at1) = y;
    }
}

template <int DT, bool HALF>
cudaError_t rotary_any(int vec, dim3 grid, cudaStream_t s, const Rows& q, uint32_t qh, const Rows& k, uint32_t kh, const Rows& qo, const Rows& ko,
                       const void* positions, int wide, const double* f, uint32_t tokens, uint32_t d, uint32_t r, float factor) {
    constexpr int W = DT == FP32 ? 4 : 8;
    return launch_early(vec ? rotary_kernel<DT, HALF, W> : rotary_kernel<DT, HALF, 1>, grid, dim3(256), 0, s, q, qh, k, kh, qo, ko, positions, wide, f, tokens, d, r,
                        factor);
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
// min / max over groups of L neighbouring lanes
template <int L>
__device__ __forceinline__ void group_range(float& lo, float& hi) {
#pragma unroll
    for (int o = 1; o < L; o *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
}

template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typename Tr<DT>::T v[2] = {Tr<DT>::from_f(a), Tr<DT>::from_f(b)};
    return *reinterpret_cast<const uint32_t*>(v);
}

// code of x in steps from lo, the nearest, ties to even, exactly as over the reals: a first guess by a product, then the two
// comparisons with its borders in exact arithmetic (difference of halves with its rounding error; border * step has 16 bits).
// Everything is halved so that the range of a bf16 group does not overflow.
__device__ __forceinline__ uint32_t code_of(float xh, float loh, float steph, float inv) {
    const float d = xh - loh;
    const float back = d + loh;                                  // two-difference: xh - loh = d + e
    const float e = (xh - back) + ((back - d) - loh);
    const float guess = inv != 0.0f ? d * inv : d / steph;
    float n = fminf(fmaxf(rintf(guess), 0.0f), 15.0f);
    const bool odd = ((int)n & 1) != 0;
    const float above = fmaf(-(n + 0.5f), steph, d) + e, below = fmaf(-(n - 0.5f), steph, d) + e;
    if (above > 0.0f || (above == 0.0f && odd)) n += 1.0f;
    else if (below < 0.0f || (below == 0.0f && odd)) n -= 1.0f;
    return (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f);
}

// Bound by memory (2 bytes an element in, half a byte out), with about 25 instructions an element beside it.  A lane takes the four
// elements of a 16-bit word of keys and of values, so 128 elements of a head are one coalesced 256-byte read of each and the group
// extremes are a few shuffles.
template <int DT, int D, int GS, bool VEC>
__global__ void __launch_bounds__(256) append_kernel(Rows k, Rows v, const void* slots, int wide, Kv4Cache c, uint32_t tokens, unsigned* err) {
    using T = typename Tr<DT>::T;
    constexpr uint32_t BL = D < 128 ? D : 128;          // elements of a unit
    constexpr uint32_t LANES = BL / 4;                   // lanes of a unit
    constexpr uint32_t UNITS = D / BL;                   // units of a head
    constexpr int GL = GS / 4;                           // lanes of a group
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t units = (uint64_t)tokens * c.kv_heads * UNITS;
    constexpr uint32_t PER_WARP = 32 / LANES;
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x / 32u);
    const uint64_t rounds = (units + PER_WARP - 1) / PER_WARP;
    for (uint64_t i = (uint64_t)blockIdx.x * (blockDim.x / 32u) + (threadIdx.x >> 5); i < rounds; i += warps) {
        const uint64_t unit = i * PER_WARP + lane / LANES;
        const bool live = unit < units;
        const uint32_t th = live ? (uint32_t)(unit / UNITS) : 0u;
        const uint32_t t = th / c.kv_heads, h = th % c.kv_heads;
        const uint32_t u = (UNITS > 1 ? (uint32_t)(unit % UNITS) * (BL / 4) : 0u) + lane % LANES;
        const long long slot = wide ? reinterpret_cast<const long long*>(slots)[t] : (long long)reinterpret_cast<const int*>(slots)[t];
        const uint32_t page_tokens = c.page_cells * kCellTokens;
        const bool inside = slot >= 0 && slot < (long long)c.pages * page_tokens;
        if (live && slot >= 0 && !inside && lane % LANES == 0u) raise_error(err, kErrKv4Page);
        const long long page = inside ? slot / page_tokens : 0;
        const uint32_t in_page = inside ? (uint32_t)(slot % page_tokens) : 0u;
        uint8_t* cell = c.data + ((size_t)page * c.kv_heads + h) * c.page_bytes + (size_t)(in_page / kCellTokens) * kv4_cell_bytes(D, GS);
        const uint32_t r = in_page % kCellTokens;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const Rows& x = side ? v : k;
            const T* src = reinterpret_cast<const T*>(x.p) + (long long)t * x.token + (long long)h * x.head + 4u * u;
            float f[4] = {0.f, 0.f, 0.f, 0.f};
            if (live) {
                if constexpr (VEC) {
                    const uint2 raw = *reinterpret_cast<const uint2*>(src);
                    const float2 a = unpack2<DT>(raw.x), b = unpack2<DT>(raw.y);
                    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[j] = Tr<DT>::to_f(src[j]);
                }
            }
            // an element that is no number makes the range of its group infinite: the group reads back as NaN
            float lo = INFINITY, hi = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool number = fabsf(f[j]) < INFINITY;
                lo = fminf(lo, number ? f[j] : -INFINITY);
                hi = fmaxf(hi, number ? f[j] : INFINITY);
            }
            group_range<GL>(lo, hi);
            float step = Tr<DT>::to_f(Tr<DT>::from_f((0.5f * hi - 0.5f * lo) / 7.5f));
            if (!(hi < INFINITY) || !(lo > -INFINITY)) { lo = __int_as_float(0x7fc00000); step = 0.0f; }
            const float steph = 0.5f * step, loh = 0.5f * lo;
            const float inv = steph >= 1e-30f ? 1.0f / steph : 0.0f;
            uint32_t word = 0;
            if (step > 0.0f) {
#pragma unroll
                for (int j = 0; j < 4; ++j) word |= code_of(0.5f * f[j], loh, steph, inv) << (4 * j);
            }
            if (live && inside) {
                *reinterpret_cast<uint16_t*>(cell + (side ? kv4_value_word(D, r, u) : kv4_key_word(D, r, u))) = (uint16_t)word;
                if (u % (GS / 4) == 0u)
                    *reinterpret_cast<uint32_t*>(cell + (side ? kv4_value_step(D, GS, r, u / (GS / 4)) : kv4_key_step(D, GS, r, u / (GS / 4)))) =
                        pack2<DT>(step, lo);
            }
        }
    }
}

// ---- rows out of the cache -----------------------------------------------------------------------------------
template <int DT, int D, int GS>
__global__ void __launch_bounds__(256) gather_kernel(Kv4Cache c, const void* slots, int wide, void* k_out, void* v_out, uint32_t tokens, unsigned* err) {
    using T = typename Tr<DT>::T;
    pdl_trigger();
    pdl_wait();
    constexpr uint32_t Q = D / 4;
    const uint64_t total = (uint64_t)tokens * c.kv_heads * Q;
    const uint32_t page_tokens = c.page_cells * kCellTokens;
    const float most = DT == FP16 ? 65504.0f : 3.38953139e38f;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t th = i / Q;
        const uint32_t u = (uint32_t)(i % Q);
        const uint32_t t = (uint32_t)(th / c.kv_heads), h = (uint32_t)(th % c.kv_heads);
        const long long slot = wide ? reinterpret_cast<const long long*>(slots)[t] : (long long)reinterpret_cast<const int*>(slots)[t];
        const bool inside = slot >= 0 && slot < (long long)c.pages * page_tokens;
        if (slot >= 0 && !inside && u == 0u) raise_error(err, kErrKv4Page);
        const long long page = inside ? slot / page_tokens : 0;
        const uint32_t in_page = inside ? (uint32_t)(slot % page_tokens) : 0u;
        const uint8_t* cell = c.data + ((size_t)page * c.kv_heads + h) * c.page_bytes + (size_t)(in_page / kCellTokens) * kv4_cell_bytes(D, GS);
        const uint32_t r = in_page % kCellTokens, g = u / (GS / 4);
        uint32_t w[2] = {0, 0}, s[2] = {0, 0};
        if (inside) {
            w[0] = *reinterpret_cast<const uint16_t*>(cell + kv4_key_word(D, r, u));
            w[1] = *reinterpret_cast<const uint16_t*>(cell + kv4_value_word(D, r, u));
            s[0] = *reinterpret_cast<const uint32_t*>(cell + kv4_key_step(D, GS, r, g));
            s[1] = *reinterpret_cast<const uint32_t*>(cell + kv4_value_step(D, GS, r, g));
        }
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const float2 st = unpack2<DT>(s[side]);
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = fmaf((float)((w[side] >> (4 * j)) & 15u), st.x, st.y);
                f[j] = x != x ? x : fminf(fmaxf(x, -most), most);      // a step is rounded: the largest code may lie above the type
            }
            T* dst = reinterpret_cast<T*>(side ? v_out : k_out) + i * 4u;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]));
        }
    }
}

template <int DT, int D, int GS>
cudaError_t run_append(const Rows& k, const Rows& v, const void* slots, int wide, const Kv4Cache& c, uint32_t tokens, bool vec, unsigned* err, cudaStream_t s) {
    constexpr uint32_t per_block = 8u * (D < 128 ? 128 / D : 1);
    const uint64_t units = (uint64_t)tokens * c.kv_heads * (D < 128 ? 1 : D / 128);
    uint64_t blocks = (units + per_block - 1) / per_block;
    const uint64_t most = (uint64_t)device_sms() * 8u;
    if (blocks > most) blocks = most;
    return launch_early(vec ? append_kernel<DT, D, GS, true> : append_kernel<DT, D, GS, false>, dim3((unsigned)blocks), dim3(256), 0, s, k, v, slots, wide, c,
                        tokens, err);
}

template <int DT, int D, int GS>
cudaError_t run_gather(const Kv4Cache& c, const void* slots, int wide, void* k, void* v, uint32_t tokens, unsigned* err, cudaStream_t s) {
    uint64_t blocks = ((uint64_t)tokens * c.kv_heads * (D / 4) + 255u) / 256u;
    const uint64_t most = (uint64_t)device_sms() * 16u;
    if (blocks > most) blocks = most;
    return launch_early(gather_kernel<DT, D, GS>, dim3((unsigned)blocks), dim3(256), 0, s, c, slots, wide, k, v, tokens, err);
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
    // a token is one block while there are tokens enough for every SM; fewer are cut by heads
    const uint32_t steps = (q_heads + k_heads) * d / (2u * (vec ? W : 1));
    uint32_t cut = (2u * device_sms() + tokens - 1u) / tokens;
    const uint32_t most = (steps + 255u) / 256u;
    if (cut > most) cut = most;
    if (cut == 0) cut = 1;
    const dim3 grid(tokens, cut);
#define ROTARY(DT_) return interleaved ? rotary_any<DT_, false>(vec, grid, s, q, q_heads, k, k_heads, qo, ko, positions, wide, f, tokens, d, r, factor) \
                                       : rotary_any<DT_, true>(vec, grid, s, q, q_heads, k, k_heads, qo, ko, positions, wide, f, tokens, d, r, factor)
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
    const bool vec = aligned(k, k_token, k_head, 4, 2) && aligned(v, v_token, v_head, 4, 2);
    return launched(for_format(dtype, head_dim, group_size, AppendCall{rk, rv, slots, slots_wide, c, tokens, vec, err, s}), "append launch");
}

int decdec_kv4_gather(const void* cache, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t group_size,
                      const void* slots, int slots_wide, uint32_t tokens, void* k_out, void* v_out, int dtype, void* stream) {
    if (int r = check_format(dtype, head_dim, group_size, page_size, cache, pages, kv_heads)) return r;
    if (tokens == 0) return 0;
    if (!k_out || !v_out || !slots) return fail(DECDEC_E_INVALID, "null pointer argument");
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 7u) return fail(DECDEC_E_INVALID, "outputs must be 8-byte aligned");
    if ((uint64_t)tokens * kv_heads > 0x7fffffffull) return fail(DECDEC_E_UNSUPPORTED, "too many rows");
    unsigned* err = nullptr;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (int r = stream_error_word(s, &err)) return r;
    const Kv4Cache c = make_cache(cache, pages, page_size, kv_heads, head_dim, group_size);
    return launched(for_format(dtype, head_dim, group_size, GatherCall{c, slots, slots_wide, k_out, v_out, tokens, err, s}), "gather launch");
}

}  // extern "C"
