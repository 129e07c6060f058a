// A key/value cache in pages for batches of requests of any lengths (ids 47..49, the fast set): the step's page tables and
// slots from the request lengths, the append of new keys and values to their slots, and the attention of the new tokens
// over their requests' pages. Lengths, tables and slots are device memory, so a recorded list replays for new ones; every
// index that comes from device memory is checked against its tensor, and every sum of lengths against its word, before it
// is used.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>
#include <vector>

#include "contract.hpp"
#include "device.hpp"
#include "fast_common.hpp"
#include "paged.hpp"

namespace lrm {

using namespace fast;

namespace {

// a + b, at most 2^32 - 1 (still associative, so a scan in any order gives the same)
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
    const uint32_t s = a + b;
    return s < a ? 0xFFFFFFFFu : s;
}

// The inclusive scan of v over the workgroup's threads; red: a word of LDS per wave, free again after the next barrier.
__device__ __forceinline__ uint32_t scan_sat(uint32_t v, uint32_t* red) {
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d, 64);
        if (lane >= d) v = add_sat(v, o);
    }
    if (lane == 63) red[wv] = v;
    __syncthreads();
    for (int i = 0; i < wv; ++i) v = add_sat(v, red[i]);
    return v;
}

// the first r with ends[r] > x (x < ends[n - 1])
__device__ __forceinline__ int first_above(const uint32_t* ends, int n, uint32_t x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (ends[m] > x)
            hi = m;
        else
            lo = m + 1;
    }
    return lo;
}

// ---------------------------------------------------------------- 47 paged_plan
// begin = min(past, blocks page), end = min(past + fresh, blocks page); request r takes ceil(end / page) - ceil(begin /
// page) pages off the free list, after those of the requests before it; row j of its fresh ones has position past + j and
// the slot of that position. Every workgroup scans the R lengths itself (two scans in LDS, at most 16 requests a thread)
// and then finds its rows' requests by bisection, so one launch does it: what bounds it is the latency of the lengths'
// load, the scans and the table's load one after the other (64 requests of one token 3.3 us, 700 requests with 25,600 rows
// 6.0 us).
__global__ __launch_bounds__(256) void k_paged_plan(const uint32_t* past, const uint32_t* fresh, const uint32_t* free,
                                                    uint32_t* table, uint32_t* starts, uint32_t* context,
                                                    uint32_t* positions, uint32_t* slots, uint32_t* counts, uint32_t R,
                                                    uint32_t blocks, uint32_t page_log2, uint32_t pages, uint32_t free_count,
                                                    uint32_t tokens) {
    __shared__ uint32_t row_end[paged::kMaxRequests];
    __shared__ uint32_t new_end[paged::kMaxRequests];
    __shared__ uint32_t red[8];
    __shared__ uint32_t over;
    const uint32_t t = threadIdx.x, page = 1u << page_log2, most = blocks * page;
    auto pages_of = [&](uint32_t n) { return (n >> page_log2) + uint32_t((n & (page - 1)) != 0); };
    auto need_of = [&](uint32_t p, uint32_t f) {
        return pages_of(min(add_sat(p, f), most)) - pages_of(min(p, most));
    };
    if (t == 0) over = 0;
    __syncthreads();
    // thread t's requests per_thread t ..
    const uint32_t per = (R + 255) / 256, r0 = min(t * per, R), r1 = min(r0 + per, R);
    uint32_t rows = 0, fills = 0, past_most = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const uint32_t p = past[r], f = fresh[r];
        rows = add_sat(rows, f);
        fills = add_sat(fills, need_of(p, f));
        past_most |= add_sat(p, f) > most;
        row_end[r] = rows;
        new_end[r] = fills;
    }
    if (past_most) over = 1;
    const uint32_t rows_end = scan_sat(rows, red), fills_end = scan_sat(fills, red + 4);
    // what the threads before this one hold (a saturated sum says nothing of its parts)
    const uint32_t rows_before = __shfl_up(rows_end, 1, 64), fills_before = __shfl_up(fills_end, 1, 64);
    uint32_t rb = rows_before, fb = fills_before;
    if ((t & 63) == 0) {
        rb = fb = 0;
        for (uint32_t i = 0; i < (t >> 6); ++i) {
            rb = add_sat(rb, red[i]);
            fb = add_sat(fb, red[4 + i]);
        }
    }
    for (uint32_t r = r0; r < r1; ++r) {
        row_end[r] = add_sat(row_end[r], rb);
        new_end[r] = add_sat(new_end[r], fb);
    }
    __syncthreads();
    const uint32_t total = row_end[R - 1], fill = new_end[R - 1];
    if (blockIdx.x == 0) {
        for (uint32_t r = t; r < R; r += 256) {
            starts[r + 1] = min(row_end[r], tokens);
            context[r] = min(add_sat(past[r], fresh[r]), most);
        }
        if (t == 0) {
            starts[0] = 0;
            counts[0] = total;
            counts[1] = fill;
            counts[2] = uint32_t(total > tokens) | over << 1 | uint32_t(fill > free_count) << 2;
        }
    }
    const uint32_t at = blockIdx.x * 256 + t, stride = gridDim.x * 256;
    for (uint32_t e = at; e < fill; e = add_sat(e, stride)) {
        const int r = first_above(new_end, int(R), e);
        const uint32_t j = e - (r ? new_end[r - 1] : 0);
        table[size_t(r) * blocks + pages_of(min(past[r], most)) + j] = e < free_count ? free[e] : paged::kNone;
    }
    const uint32_t valid = min(total, tokens);
    for (uint32_t i = at; i < valid; i = add_sat(i, stride)) {
        const int r = first_above(row_end, int(R), i);
        const uint64_t pos = uint64_t(past[r]) + (i - (r ? row_end[r - 1] : 0));
        uint32_t slot = paged::kNone;
        if (pos < most) {
            const uint32_t b = uint32_t(pos) >> page_log2, have = pages_of(min(past[r], most));
            uint32_t id = paged::kNone;
            if (b < have) {
                id = table[size_t(r) * blocks + b];
            } else {
                const uint32_t e = (r ? new_end[r - 1] : 0) + (b - have);
                if (e < free_count) id = free[e];
            }
            if (id < pages) slot = (id << page_log2) + (uint32_t(pos) & (page - 1));
        }
        positions[i] = uint32_t(pos);
        slots[i] = slot;
    }
}

// ---------------------------------------------------------------- element types

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float widen<_Float16>(_Float16 v) {
    return static_cast<float>(v);
}
template <>
__device__ __forceinline__ float widen<__bf16>(__bf16 v) {
    return bf2f(__builtin_bit_cast(uint16_t, v));
}
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ _Float16 narrow<_Float16>(float v) {
    return static_cast<_Float16>(v);
}
template <>
__device__ __forceinline__ __bf16 narrow<__bf16>(float v) {
    return __builtin_bit_cast(__bf16, f2bf(v));
}

// two floats to a pair of the type, round to nearest even (one conversion instruction)
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, t2));
}

// Two results of the attention to a pair of the type. A result is a mean of the values, but its weights' rounding may put it up
// to 2^-11 past them, and next to fp16's end past that: it ends there too (an infinity comes from the values and stays).
template <typename T>
__device__ __forceinline__ uint32_t pack_mean(float a, float b) {
    if constexpr (std::is_same_v<T, _Float16>) {
        constexpr float end = 65504.f;
        a = fabsf(a) < INFINITY ? __builtin_amdgcn_fmed3f(a, -end, end) : a;
        b = fabsf(b) < INFINITY ? __builtin_amdgcn_fmed3f(b, -end, end) : b;
    }
    return pack<T>(a, b);
}

// N consecutive elements as floats, in one load
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = widen<T>(x[i]);
}
// N consecutive floats narrowed, in one store
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float (&v)[N]) {
    typedef uint32_t vec __attribute__((ext_vector_type(N / 2)));
    vec x;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) x[i] = pack<T>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<vec*>(p) = x;
}

// the sum over the N lanes of an aligned group
template <int N>
__device__ __forceinline__ float sum_lanes(float v) {
    v = quad4_sum(v);
    if constexpr (N >= 8) v += dpp_f<0x141>(v);
    if constexpr (N >= 16) v += dpp_f<0x140>(v);
    return v;
}

// ---------------------------------------------------------------- 48 qk_norm_rope_append_paged
// n = w x / sqrt(mean x^2 + eps) over a head, (a, b) its halves: (a cos - b sin, b cos + a sin) at the row's position; values
// as they are. Everything is float32 until the one rounding to the cache's type (nearest even) at the stores.
// Values past fp16's range become infinities, as its rounding has it. Bound by the projections' bytes (9,200 rows of
// 32 + 8 + 8 heads of 128 in bf16: 47 us, 5.2 TB/s, back to back; 512 rows 5.2 us, the latency of three loads that wait for each
// other). Queries and keys: a head is 4 to 16 lanes with 16 bytes of its lower and of its upper half each, so a lane holds the pairs that the rotation turns, the sum of squares is a few DPP adds, and a wave takes 4 to
// 16 heads of a row at a time; the row's rotation and the norm weights are loaded once per wave. Values: a wave takes the
// runs of rows that begin in its 8 rows, a run being rows whose slots follow each other in one tile of 8 positions; a
// whole run's 8 rows of a dim are one 16-byte store, and shorter runs (a single token, the ends of a chunk) store each value
// alone. Rows whose slot or position has no place are not appended.
template <typename IN, typename T, int HD>
__global__ __launch_bounds__(256) void k_paged_append(const IN* qkv, const uint16_t* qn, const uint16_t* kn,
                                                      const float* cos_t, const float* sin_t, const uint32_t* starts,
                                                      const uint32_t* positions, const uint32_t* slots, T* q, T* kc, T* vc,
                                                      uint32_t requests, uint32_t tokens, uint32_t qh, uint32_t kvh,
                                                      uint32_t max_pos, uint32_t page_log2, uint32_t pages, float eps,
                                                      uint32_t qk_blocks, uint32_t parts, uint32_t v_chunks) {
    constexpr int H = HD / 2, VEC = 16 / int(sizeof(IN)), LPH = H / VEC, HPW = 64 / LPH;
    const uint32_t lane = threadIdx.x & 63, page_mask = (1u << page_log2) - 1, w = qh + 2 * kvh;
    const uint32_t rows = min(starts[requests], tokens);
    auto place = [&](uint32_t slot, uint32_t pos) { return (slot >> page_log2) < pages && pos < max_pos; };
    const uint32_t block = blockIdx.y * gridDim.x + blockIdx.x;  // (a grid past 65,535 is folded)
    if (block < qk_blocks) {
        const uint32_t wave = block * 4 + uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
        const uint32_t row = wave / parts, part = wave % parts;
        if (row >= rows) return;
        const uint32_t pos = positions[row], slot = slots[row], heads = qh + kvh, sub = lane % LPH;
        const bool turn = pos < max_pos, keep = place(slot, pos);
        const size_t angle = size_t(turn ? pos : 0) * H + VEC * sub;
        float c[VEC], s[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            load_n(cos_t + angle + i, *reinterpret_cast<float(*)[4]>(c + i));
            load_n(sin_t + angle + i, *reinterpret_cast<float(*)[4]>(s + i));
        }
        typedef uint16_t wvec __attribute__((ext_vector_type(VEC)));
        const wvec q0 = *reinterpret_cast<const wvec*>(qn + VEC * sub), q1 = *reinterpret_cast<const wvec*>(qn + H + VEC * sub);
        const wvec k0 = *reinterpret_cast<const wvec*>(kn + VEC * sub), k1 = *reinterpret_cast<const wvec*>(kn + H + VEC * sub);
        const IN* x = qkv + size_t(row) * w * HD + VEC * sub;
        T* const krow = kc + ((size_t(slot >> page_log2) * kvh << page_log2) + (slot & page_mask)) * HD + VEC * sub;
#pragma unroll 2
        for (uint32_t head = part * HPW + lane / LPH; head < heads; head += parts * HPW) {
            float a[VEC], b[VEC];
            load_n(x + size_t(head) * HD, a);
            load_n(x + size_t(head) * HD + H, b);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
            const float r = 1.0f / sqrtf(sum_lanes<LPH>(sum) / float(HD) + eps);
            float lo[VEC], hi[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float an = bf2f(head < qh ? q0[i] : k0[i]) * (a[i] * r), bn = bf2f(head < qh ? q1[i] : k1[i]) * (b[i] * r);
                lo[i] = turn ? an * c[i] - bn * s[i] : 0.f;
                hi[i] = turn ? bn * c[i] + an * s[i] : 0.f;
            }
            if (head < qh) {
                T* y = q + (size_t(row) * qh + head) * HD + VEC * sub;
                store_n(y, lo);
                store_n(y + H, hi);
            } else if (keep) {
                T* y = krow + (size_t(head - qh) << page_log2) * HD;
                store_n(y, lo);
                store_n(y + H, hi);
            }
        }
        return;
    }
    // ---- values: 8 rows and 128 elements of the row's value heads per wave
    constexpr int E = 2;
    const uint32_t wave = (block - qk_blocks) * 4 + uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    const uint32_t row0 = wave / v_chunks * 8, flat = (wave % v_chunks) * (64 * E) + E * lane;
    if (row0 >= rows) return;
    // lane i looks at row row0 - 1 + i: does it go on where the row before it stood, in the same tile?
    const uint32_t mine = row0 + lane - 1;  // (row0 = 0, lane 0: past every row)
    const bool there = lane < 16 && mine < rows;
    const uint32_t slot = there ? slots[mine] : paged::kNone;
    const bool good = there && place(slot, positions[mine]);
    const uint32_t before = uint32_t(__shfl_up(int(slot), 1, 64));
    const uint32_t goods = uint32_t(__ballot(good)) & 0xFFFFu;
    const bool goes_on = good && lane > 0 && (goods >> (lane - 1) & 1u) && slot == before + 1 && (slot & 7) != 0;
    const uint32_t on = uint32_t(__ballot(goes_on)) & 0xFFFFu;
    uint32_t firsts = goods & ~on & 0x1FEu;  // runs that begin in this wave's rows, bit i for row0 - 1 + i
    const uint32_t head = flat / HD, dim = flat % HD;
    while (firsts) {
        const int i = __builtin_ctz(firsts);
        firsts &= firsts - 1;
        const int n = 1 + __builtin_ctz(~(on >> (i + 1)));  // rows of the run, at most 8: a tile ends it
        const uint32_t first = row0 + i - 1, at = uint32_t(__builtin_amdgcn_readlane(int(slot), i));
        if (head >= kvh) continue;
        const IN* x = qkv + (size_t(first) * w + qh + kvh) * HD + flat;
        T* y = vc + ((size_t(at >> page_log2) * kvh + head) << page_log2) * HD + size_t((at & page_mask) >> 3) * (8 * HD) + dim * 8;
        float v[8][E];
        if (n == 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) load_n(x + size_t(j) * w * HD, v[j]);
#pragma unroll
            for (int e = 0; e < E; ++e)
                *reinterpret_cast<u32x4*>(y + 8 * e) = u32x4{pack<T>(v[0][e], v[1][e]), pack<T>(v[2][e], v[3][e]),
                                                             pack<T>(v[4][e], v[5][e]), pack<T>(v[6][e], v[7][e])};
        } else {
            for (int j = 0; j < n; ++j) {
                load_n(x + size_t(j) * w * HD, v[0]);
#pragma unroll
                for (int e = 0; e < E; ++e) y[8 * e + (at & 7) + j] = narrow<T>(v[0][e]);
            }
        }
    }
}

// ---------------------------------------------------------------- 49 attention_paged
struct AttnArgs {
    const void *q, *kc, *vc;
    const uint32_t *table, *starts, *context;
    void* y;
    uint32_t* ws;
    uint32_t requests, tokens, max_fresh, qh, kvh, blocks, page_log2, pages;
    uint32_t join_here;  // the tiles' last workgroup of an item joins its parts
    float scale_log2;  // the scale times log2(e): weights are 2^(s scale_log2 - m scale_log2)
};

// A request as its lengths on the device give it, clamped to the tensors.
struct Request {
    int row0;  // its first row
    int rows;  // the rows that this dispatch computes
    int seen;  // the keys that row 0 sees; row i sees i more (below 1: none)
};
__device__ __forceinline__ Request request_of(const AttnArgs& a, uint32_t r) {
    const uint32_t s0 = min(a.starts[r], a.tokens), s1 = min(a.starts[r + 1], a.tokens);
    const int fresh = s1 > s0 ? int(s1 - s0) : 0, ctx = int(min(a.context[r], a.blocks << a.page_log2));
    return Request{int(s0), min(fresh, int(a.max_fresh)), ctx - fresh + 1};
}

// The sums of a request's share of the work over the requests before it hold because their rows lie one after the other: at
// most `tokens` in all, which is what a dispatch was checked for. Where starts decrease, the rows of several requests may
// overlap and their sums pass 32 bits, so such a sum is kNoSum from there on (add_sat and scan_sat stay there) and nothing
// is computed.
constexpr uint32_t kNoSum = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t add_share(const AttnArgs& a, uint32_t r, uint32_t sum, uint32_t share) {
    return a.starts[r + 1] < a.starts[r] ? kNoSum : add_sat(sum, share);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// words that no launch writes while it reads them, at uniform addresses: scalar loads
typedef const __attribute__((address_space(4))) uint32_t* const_words;

template <typename T>
struct Mfma;
template <>
struct Mfma<_Float16> {
    typedef f16x8 vec;
    static __device__ __forceinline__ f32x4 m16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 m32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
    }
};
template <>
struct Mfma<__bf16> {
    typedef bf16x8 vec;
    static __device__ __forceinline__ f32x4 m16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 m32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
    }
};

// Partials pass between workgroups, which may run on other XCDs: stores that go through to memory and loads that do not take
// an older line from the XCD's L2 (device scope), 16 or 8 bytes each and as many under way as there are registers (the
// atomic loads of that scope are waited for one by one: a join of two parts took 25 us, of 32 parts 320).
constexpr int kDeviceScope = 16;  // the sc1 bit of a buffer instruction
template <int SCOPE = kDeviceScope>
__device__ __forceinline__ void store_part(__amdgpu_buffer_rsrc_t r, int word, f32x4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, word * 4, 0, SCOPE);
}
template <int SCOPE = kDeviceScope>
__device__ __forceinline__ f32x4 load_part(__amdgpu_buffer_rsrc_t r, int word) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, word * 4, 0, SCOPE));
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int SCOPE = kDeviceScope>
__device__ __forceinline__ void store_part2(__amdgpu_buffer_rsrc_t r, int word, float a, float b) {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(a), __float_as_uint(b)}, r, word * 4, 0, SCOPE);
}
template <int SCOPE = kDeviceScope>
__device__ __forceinline__ float2 load_part2(__amdgpu_buffer_rsrc_t r, int word) {
    const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, word * 4, 0, SCOPE));
    return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Weights go into their product with the values rounded to the cache's type, relative to a reference that the largest may
// exceed by 2^8. fp16 ends at 2^-24, which tens of thousands of small weights behind a few large ones would fall below (64,000 of
// 2^-25 together are 0.002 of the largest), so they are 2^kUp of what they are: at most 2^15, and lost below 2^-32.
// Their sum is formed from the same, so the results are not changed otherwise.
template <typename T>
constexpr float kUp = std::is_same_v<T, _Float16> ? 7.f : 0.f;

// Values that are no finite numbers, at keys that one column of a tile sees and another does not: zero times such a value is
// NaN, so they are taken out of the product and added to the columns that see them alone. A second product with 0 / 1
// weights counts them: infinity as 1, minus infinity as 128, NaN as both; fewer than 128 keys, so float32 holds the counts.
template <typename T>
constexpr uint32_t kExponent = std::is_same_v<T, __bf16> ? 0x7F80u : 0x7C00u;
template <typename T>
__device__ __forceinline__ bool take_odd(u32x4& v) {  // zeroes them; whether there were any
    constexpr uint32_t lo = kExponent<T>, hi = lo << 16;
    bool any = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool l = (v[e] & lo) == lo, h = (v[e] & hi) == hi;
        v[e] &= (l ? 0u : 0x0000FFFFu) | (h ? 0u : 0xFFFF0000u);
        any = any || l || h;
    }
    return any;
}
template <typename T>
__device__ __forceinline__ u32x4 odd_codes(u32x4 v) {
    constexpr uint32_t exp = kExponent<T>;
    auto code = [](uint32_t x) {
        return (x & exp) != exp ? 0.f : (x & (0x7FFFu ^ exp)) ? 129.f : (x & 0x8000u) ? 128.f : 1.f;
    };
    u32x4 c;
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = pack<T>(code(v[e] & 0xFFFFu), code(v[e] >> 16));
    return c;
}
__device__ __forceinline__ float add_odd(float o, float count) {
    const uint32_t n = uint32_t(count);
    if (n & 127u) o += INFINITY;
    if (n >> 7) o -= INFINITY;
    return o;
}

// Rows of few query columns: up to 16 per request and KV head (column c = row c / group, head c % group of the KV head's).
// y = sum_k 2^((s_k - m) c) v_k / sum_k 2^((s_k - m) c) over the keys that a column sees, c the scale times log2 e, in one pass
// with a running reference m.
// Bound by the cache's bytes, so every wave streams its own keys straight into the registers that the matrix
// instruction reads (no LDS, no barrier), two units in flight, and the four waves of a workgroup meet once per item. All
// units are shared out evenly over 512 workgroups, so a long context spreads over the GPU and a batch of uneven ones leaves no
// CU behind; the last part of an item to arrive joins its partials. Measured, calls back to back on three streams: 200
// requests of up to 4000 positions 262 us, 16 of 8192 88 us (both 6.1 TB/s), one of 65,701 47 us (5.7 TB/s); single dispatches
// after a pause, at lower clocks: 287, 101 and 65 us, one of 700 8.6.
//
// A unit is 128 keys of an item, 32 per wave. S^T = K Q^T on 16 x 16 x 32 tiles: the two tiles' rows i hold the keys
// 8 (i / 4) + 4 tile + i % 4, so that lane group g = lane / 16 gets the scores of the eight keys 8 g .. 8 g + 7 of its column:
// exactly the operand that O^T = V^T P^T wants from it, with V's operand one 16-byte read of eight positions of a dim.
// No value crosses lanes but the maximum. Keys that no column sees and pages that are none are read past the buffer's
// end, which gives zeros without an access.
template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void k_attn_rows(AttnArgs a, uint32_t k_bytes, uint32_t v_bytes) {
    using M = Mfma<T>;
    constexpr int KS = HD / 32, DT = HD / 16, XR = HD + 4;  // dim steps, dim tiles, padded row of the exchange
    constexpr uint32_t kOut = 0x80000000u;                   // an offset past every buffer
    __shared__ uint32_t ends[paged::kMaxRequests];           // units of the requests up to and with r
    __shared__ __attribute__((aligned(16))) float xo[4 * 16 * XR];
    __shared__ float xm[4][16], xl[4][16];
    __shared__ uint32_t red[4];
    __shared__ uint32_t arrived;
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, c16 = lane & 15, g = lane >> 4;
    const int group = int(a.qh / a.kvh), kvh = int(a.kvh);
    const uint32_t page_mask = (1u << a.page_log2) - 1;

    // ---- the units of every request, and this workgroup's
    auto units_of = [&](const Request& q) {  // of one item of the request
        if (q.rows < 1) return 0;
        return max(1, (q.seen + q.rows - 1 + int(paged::kRowsKeys) - 1) / int(paged::kRowsKeys));
    };
    {
        const uint32_t per = (a.requests + 255) / 256, r0 = min(t * per, a.requests), r1 = min(r0 + per, a.requests);
        uint32_t sum = 0;
        for (uint32_t r = r0; r < r1; ++r) {
            sum = add_share(a, r, sum, uint32_t(units_of(request_of(a, r)) * kvh));
            ends[r] = sum;
        }
        const uint32_t before = scan_sat(sum, red) - sum;
        for (uint32_t r = r0; r < r1; ++r) ends[r] += before;
        __syncthreads();
    }
    const uint32_t total = ends[a.requests - 1], G = min(uint32_t(gridDim.x), total), w = blockIdx.x;
    if (w >= G || total == kNoSum) return;
    auto first_unit = [&](uint32_t i) { return uint32_t(uint64_t(total) * i / G); };
    auto group_of = [&](uint32_t u) { return uint32_t(((uint64_t(u) + 1) * G - 1) / total); };
    const uint32_t u0 = first_unit(w), u1 = first_unit(w + 1);

    // ---- a unit's place: request, KV head, key block
    struct Place {
        int r, h, k, n;       // unit k of the item's n
        int row0, cols, keys; // the item's first row, its columns, the keys that its last row sees
        int seen;             // the keys that its first row sees
    };
    auto enter = [&](Place& p, int r) {
        const Request q = request_of(a, uint32_t(r));
        p.r = r, p.n = uniform(units_of(q)), p.row0 = uniform(q.row0), p.cols = uniform(q.rows * group);
        p.seen = uniform(q.seen), p.keys = uniform(max(0, q.seen + q.rows - 1));
    };
    auto next = [&](Place& p) {
        if (++p.k < p.n) return;
        p.k = 0;
        if (++p.h < kvh) return;
        p.h = 0;
        int r = p.r + 1;
        while (r < int(a.requests) - 1 && uniform(int(ends[r])) == uniform(int(ends[r - 1]))) ++r;
        if (r < int(a.requests)) enter(p, r);  // past the last request the place is not used
    };
    Place p0{};
    {
        const int r = uniform(first_above(ends, int(a.requests), u0));
        enter(p0, r);
        const uint32_t in = u0 - (r ? uint32_t(uniform(int(ends[r - 1]))) : 0u);
        p0.h = int(in) / p0.n, p0.k = int(in) % p0.n;
    }

    const __amdgpu_buffer_rsrc_t k_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.kc), 0, k_bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t v_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.vc), 0, v_bytes, 0x00020000);
    // this wave's keys of a unit start at 128 k + 32 wv; this lane's K rows of both tiles lie in the eight from 8 (c16 / 4),
    // its V reads take the eight from 8 g
    const int k8 = 32 * wv + 8 * (c16 >> 2), v8 = 32 * wv + 8 * g;
    auto page_ids = [&](const Place& p, uint32_t& idk, uint32_t& idv) {
        const uint32_t* row = a.table + size_t(p.r) * a.blocks;
        const uint32_t kb = uint32_t(p.k) * paged::kRowsKeys;
        idk = row[min((kb + k8) >> a.page_log2, a.blocks - 1)];
        idv = row[min((kb + v8) >> a.page_log2, a.blocks - 1)];
    };
    u32x4 kr[2][2 * KS], vr[2][DT];
    bool page_in[2];  // this lane's eight keys have a page
    auto fetch = [&](auto set, const Place& p, uint32_t idk, uint32_t idv) __attribute__((always_inline)) {
        constexpr int S = decltype(set)::value;
        const int kk = p.k * int(paged::kRowsKeys) + k8, kv = p.k * int(paged::kRowsKeys) + v8;
        const bool ink = kk < p.keys && idk < a.pages, inv = kv < p.keys && idv < a.pages;
        page_in[S] = idv < a.pages;
        const uint32_t ko = ink ? ((((idk * uint32_t(kvh) + p.h) << a.page_log2) + (uint32_t(kk) & page_mask) + (c16 & 3)) * HD +
                                   8 * g) * 2
                                : kOut;
        const uint32_t vo = inv ? ((((idv * uint32_t(kvh) + p.h) << a.page_log2) + (uint32_t(kv) & page_mask)) * HD + 8 * c16) * 2
                                : kOut;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                kr[S][i * KS + s] = __builtin_amdgcn_raw_buffer_load_b128(k_rsrc, ko + i * 8 * HD + s * 64, 0, 0);
#pragma unroll
        for (int d = 0; d < DT; ++d) vr[S][d] = __builtin_amdgcn_raw_buffer_load_b128(v_rsrc, vo + d * 256, 0, 0);
    };
    u32x4 qf[KS], qn[KS];
    auto fetch_q = [&](const Place& p) __attribute__((always_inline)) {
        const int row = p.row0 + c16 / group, head = p.h * group + c16 % group;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qn[s] = u32x4{0u, 0u, 0u, 0u};
            if (c16 < p.cols)
                qn[s] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + (size_t(row) * a.qh + head) * HD + 32 * s +
                                                        8 * g);
        }
    };

    float m_run = -INFINITY, l_run = 0.f;  // the column's reference maximum, this lane's share of its sum
    f32x4 o[DT];
    auto clear = [&]() __attribute__((always_inline)) {
        m_run = -INFINITY, l_run = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    auto compute = [&](auto set, const Place& p) __attribute__((always_inline)) {
        constexpr int S = decltype(set)::value;
        const int kb = p.k * int(paged::kRowsKeys) + 32 * wv;  // this wave's first key
        f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            s0 = M::m16(kr[S][s], qf[s], s0);
            s1 = M::m16(kr[S][KS + s], qf[s], s1);
        }
        bool odd = false;  // some value that not all columns see is no finite number
        float sc[8];  // keys kb + 8 g ..
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] = s0[e], sc[4 + e] = s1[e];
        if (kb + 32 > p.seen || __any(!page_in[S])) {  // uniform: some key is hidden from some column
            const int lim = page_in[S] && c16 < p.cols ? p.seen + c16 / group - kb - 8 * g : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) sc[e] = e < lim ? sc[e] : -INFINITY;
            if (kb + 32 > p.keys) {  // what lies past the last key may be anything, and zero times NaN is NaN
                const int left = p.keys - kb - 8 * g;
                u32x4 keep;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    keep[e] = (2 * e < left ? 0x0000FFFFu : 0u) | (2 * e + 1 < left ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int d = 0; d < DT; ++d) vr[S][d] &= keep;
            }
            if (p.keys > p.seen) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    u32x4 x = vr[S][d];
                    odd |= take_odd<T>(x);
                }
                odd = __any(odd);
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
        mx = cross_rows_max(mx);
        // the reference moves only when it is left behind by more than 8 in the exponent: weights stay at most 2^8
        const bool grow = (mx - m_run) * a.scale_log2 > 8.0f;  // false for NaN (both -inf)
        if (__any(grow)) {
            const float alpha = grow ? __builtin_amdgcn_exp2f((m_run - mx) * a.scale_log2) : 1.0f;
            m_run = grow ? mx : m_run;
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= alpha;
        }
        const float mc = m_run == -INFINITY ? 0.f : m_run * a.scale_log2 - kUp<T>;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], a.scale_log2, -mc));
            l_run += sc[e];
        }
        // the weights go into the product rounded to the cache's type, as its values are; their sum stays float32
        const u32x4 pb = {pack<T>(sc[0], sc[1]), pack<T>(sc[2], sc[3]), pack<T>(sc[4], sc[5]), pack<T>(sc[6], sc[7])};
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (odd) {
                const int lim = p.seen + c16 / group - kb - 8 * g;
                u32x4 sees;
#pragma unroll
                for (int e = 0; e < 4; ++e) sees[e] = pack<T>(2 * e < lim ? 1.f : 0.f, 2 * e + 1 < lim ? 1.f : 0.f);
                const f32x4 counts = M::m16(odd_codes<T>(vr[S][d]), sees, f32x4{0.f, 0.f, 0.f, 0.f});
                take_odd<T>(vr[S][d]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][e] = add_odd(o[d][e], counts[e]);
            }
            o[d] = M::m16(vr[S][d], pb, o[d]);
        }
    };

    // ---- the end of an item here: the waves' parts meet in LDS, then y, or a partial and the join
    auto add_part = [&](float& m, float& sum, f32x4& v, float mo, float so, f32x4 vo) __attribute__((always_inline)) {
        const float mn = fmaxf(m, mo), mc = mn == -INFINITY ? 0.f : mn * a.scale_log2;
        const float fo = __builtin_amdgcn_exp2f(m * a.scale_log2 - mc), fn = __builtin_amdgcn_exp2f(mo * a.scale_log2 - mc);
        sum = sum * fo + so * fn;
        v = v * fo + vo * fn;
        m = mn;
    };
    constexpr int SW = int(paged::slot_words(paged::kRowsCols, HD));
    const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc(
        a.ws, 0, int(4 * (paged::kGroups + 2 * paged::kRowsGroups * SW)), 0x00020000);
    auto slot_at = [&](uint32_t i, bool begins) { return int(paged::kGroups) + int(2 * i + (begins ? 1 : 0)) * SW; };
    auto finish = [&](const Place& p, uint32_t u) {
        const float l = cross_rows_sum(l_run);
        if (g == 0) xm[wv][c16] = m_run, xl[wv][c16] = l;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(xo + (wv * 16 + c16) * XR + 16 * d + 4 * g) = o[d];
        lds_barrier();
        // thread t: four dims of column t / (HD / 4) + i 1024 / HD
        const uint32_t begin = u - uint32_t(p.k), end = begin + uint32_t(p.n);
        const bool whole = begin >= u0 && end <= u1;
        const uint32_t wa = group_of(begin), wb = group_of(end - 1);
        const int mine = slot_at(w, begin >= u0);
        constexpr int Q4 = HD / 4;
        for (int e = t; e < p.cols * Q4; e += 256) {
            const int c = e / Q4, d = 4 * (e % Q4);
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, xm[i][c]);
            const float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
            float sum = 0.f;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = __builtin_amdgcn_exp2f(xm[i][c] * a.scale_log2 - mc);
                sum = fmaf(xl[i][c], f, sum);
                v += *reinterpret_cast<const f32x4*>(xo + (i * 16 + c) * XR + d) * f;
            }
            if (whole) {
                const float inv = sum != 0.f ? 1.0f / sum : 0.f;  // no key at all: zeros
                const int row = p.row0 + c / group, head = p.h * group + c % group;
                T* y = static_cast<T*>(a.y) + (size_t(row) * a.qh + head) * HD + d;
                *reinterpret_cast<uint2*>(y) = make_uint2(pack_mean<T>(v[0] * inv, v[1] * inv), pack_mean<T>(v[2] * inv, v[3] * inv));
            } else {
                store_part(ws, mine + 2 * int(paged::kRowsCols) + c * HD + d, v);
                if (d == 0) store_part2(ws, mine + 2 * c, m, sum);
            }
        }
        if (!whole) {
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0): this wave's stores are performed
            lds_barrier();
            uint32_t* counter = a.ws + wa;
            if (t == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            lds_barrier();
            if (arrived == wb - wa) {  // the last one in joins the parts, in their order
                // a thread takes four dims of a column over the parts wa + k, wa + k + K, ..: K threads share a column's
                // dims where there are that many, and meet in LDS
                const int lanes = p.cols * Q4, share = lanes >= 256 ? 1 : 256 / lanes;
                for (int e0 = 0; e0 < lanes; e0 += 256) {
                    const int e = share > 1 ? t % lanes : e0 + t, k = share > 1 ? t / lanes : 0;
                    const int c = e / Q4, d = 4 * (e % Q4);
                    float m = -INFINITY, sum = 0.f;
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
                    if (e < lanes && k < share) {
                        constexpr int PF = 6;
                        for (uint32_t i = wa + k; i <= wb; i += PF * share) {
                            float2 ml[PF];
                            f32x4 x[PF];
#pragma unroll
                            for (int q = 0; q < PF; ++q) {
                                const uint32_t part = min(i + q * share, wb);
                                const int at = slot_at(part, part == wa);
                                ml[q] = load_part2(ws, at + 2 * c);
                                x[q] = load_part(ws, at + 2 * int(paged::kRowsCols) + c * HD + d);
                            }
#pragma unroll
                            for (int q = 0; q < PF; ++q) {
                                if (i + q * share > wb) continue;
                                add_part(m, sum, v, ml[q].x, ml[q].y, x[q]);
                            }
                        }
                    }
                    if (share > 1) {
                        float* const mine = xo + t * 8;
                        *reinterpret_cast<f32x4*>(mine) = v;
                        mine[4] = m, mine[5] = sum;
                        lds_barrier();
                        if (t < lanes)
                            for (int j = 1; j < share; ++j) {
                                const float* other = xo + (t + j * lanes) * 8;
                                add_part(m, sum, v, other[4], other[5], *reinterpret_cast<const f32x4*>(other));
                            }
                    }
                    if (e < lanes && k == 0) {
                        const float inv = sum != 0.f ? 1.0f / sum : 0.f;
                        const int row = p.row0 + c / group, head = p.h * group + c % group;
                        T* y = static_cast<T*>(a.y) + (size_t(row) * a.qh + head) * HD + d;
                        *reinterpret_cast<uint2*>(y) =
                            make_uint2(pack_mean<T>(v[0] * inv, v[1] * inv), pack_mean<T>(v[2] * inv, v[3] * inv));
                    }
                }
                if (t == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        lds_barrier();  // the exchange is free again
        clear();
    };

    // ---- the units: page ids two ahead, keys and values one ahead of the products
    using A0 = std::integral_constant<int, 0>;
    using A1 = std::integral_constant<int, 1>;
    Place p1 = p0, p2 = p0;
    uint32_t idk = 0, idv = 0, idk1 = 0, idv1 = 0;
    page_ids(p0, idk, idv);
    fetch_q(p0);
    next(p1);
    p2 = p1;
    if (u0 + 1 < u1) page_ids(p1, idk1, idv1);
    fetch(A0{}, p0, idk, idv);
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = qn[s];
    clear();
    auto step = [&](auto set, uint32_t u) __attribute__((always_inline)) {
        constexpr int S = decltype(set)::value;
        using N = std::integral_constant<int, 1 - S>;
        // p0 is unit u, p1 unit u + 1 with its ids in idk1, idv1
        const bool more = u + 1 < u1, item = more && p1.k == 0;
        idk = idk1, idv = idv1;
        if (u + 2 < u1) {
            next(p2);
            page_ids(p2, idk1, idv1);
        }
        if (more) {
            if (item) fetch_q(p1);
            fetch(N{}, p1, idk, idv);
        }
        __builtin_amdgcn_sched_barrier(0);
        compute(set, p0);
        if (!more || item) finish(p0, u);
        if (item) {
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] = qn[s];
        }
        p0 = p1, p1 = p2;
    };
    for (uint32_t u = u0; u < u1; u += 2) {
        step(A0{}, u);
        if (u + 1 >= u1) break;
        step(A1{}, u + 1);
    }
}

// sum over i < n of floor((b + i step) / 64) (Euclid's way down the two slopes), for sums below 2^31
__device__ __forceinline__ uint32_t floor_sum64(uint32_t n, uint32_t step, uint32_t b) {
    // the first step, whose divisor is known
    uint32_t sum = uint32_t(uint64_t(n) * (n - 1) / 2) * (step / 64) + n * (b / 64), m = 64;
    step %= 64, b %= 64;
    const uint32_t y0 = step * n + b;
    n = y0 / 64, b = y0 % 64;
    const uint32_t s0 = step;
    step = m, m = s0;
    while (n) {
        sum += uint32_t(uint64_t(n) * (n - 1) / 2) * (step / m) + n * (b / m);
        step %= m, b %= m;
        const uint32_t y = step * n + b;
        n = y / m, b = y % m;
        const uint32_t s = step;
        step = m, m = s;
        if (!m) break;
    }
    return sum;
}

// The join of an item of the tiles: y = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over its parts, in their order. This wave
// takes a quarter part_d of the dims of its 32 columns of the tile.
struct Split {
    int parts, base, stride, first;  // part i in slot base + i stride (+ `first` for the first)
    int row0, cols, hk;
};
template <typename T, int HD, int NW, int SCOPE>
__device__ __forceinline__ void join_item(const AttnArgs& a, const Split& p, int wv, int part_d, int lane) {
    constexpr int DT = HD / 32, N = DT;  // 16 bytes per lane and part
    constexpr uint32_t GROUPS = paged::tile_groups(NW), COLS = paged::tile_cols(NW), SLOTS = paged::tile_slots(NW);
    constexpr int SW = int(paged::slot_words(COLS, HD));
    const int parts = p.parts, cols = p.cols, row0 = p.row0, hk = p.hk, col = 32 * wv + (lane & 31);
    const __amdgpu_buffer_rsrc_t ws =
        __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, int(4 * (SLOTS + 2 * GROUPS * SW)), 0x00020000);
    auto slot_at = [&](int i) { return int(SLOTS) + (p.base + i * p.stride + (i ? 0 : p.first)) * SW; };
    constexpr int PF = SCOPE ? 2 : 6;  // parts under way (the tiles have fewer registers to spare)
    float top = -INFINITY, l = 0.f, sum[4 * N];
#pragma unroll
    for (int e = 0; e < 4 * N; ++e) sum[e] = 0.f;
    for (int i = 0; i < parts; i += PF) {
        float2 ml[PF];
        f32x4 x[PF][N];
#pragma unroll
        for (int q = 0; q < PF; ++q) {
            if (i + q >= parts) break;
            const int slot = slot_at(i + q);
            ml[q] = load_part2<SCOPE>(ws, slot + 2 * col);
#pragma unroll
            for (int j = 0; j < N; ++j)
                x[q][j] = load_part<SCOPE>(ws, slot + 2 * int(COLS) + ((wv * 4 * DT + part_d * N + j) * 64 + lane) * 4);
        }
        __builtin_amdgcn_sched_barrier(0);  // (all under way before the first is waited for)
        float most = top;
#pragma unroll
        for (int q = 0; q < PF; ++q) {
            if (i + q >= parts) break;
            most = fmaxf(most, ml[q].x);
        }
        const float tc = most == -INFINITY ? 0.f : most * a.scale_log2;
        const float back = __builtin_amdgcn_exp2f(top * a.scale_log2 - tc);
        top = most;
        l *= back;
#pragma unroll
        for (int e = 0; e < 4 * N; ++e) sum[e] *= back;
#pragma unroll
        for (int q = 0; q < PF; ++q) {
            if (i + q >= parts) break;
            const float f = __builtin_amdgcn_exp2f(ml[q].x * a.scale_log2 - tc);
            l += ml[q].y * f;
#pragma unroll
            for (int e = 0; e < 4 * N; ++e) sum[e] += x[q][e >> 2][e & 3] * f;
        }
    }
    if (col >= cols) return;
    const int group = int(a.qh / a.kvh);
    const float inv = l != 0.f ? 1.0f / l : 0.f;  // no key at all: zeros
    T* y = static_cast<T*>(a.y) + (size_t(row0 + col / group) * a.qh + hk * group + col % group) * HD + 4 * (lane >> 5);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int i = part_d * N + j;  // dims 32 (i / 4) + 8 (i % 4) + 4 h ..
        *reinterpret_cast<uint2*>(y + 32 * (i >> 2) + 8 * (i & 3)) =
            make_uint2(pack_mean<T>(sum[4 * j] * inv, sum[4 * j + 1] * inv), pack_mean<T>(sum[4 * j + 2] * inv, sum[4 * j + 3] * inv));
    }
}

// Rows of many query columns, on 32 x 32 x 16 tiles. A tile of an item is up to 32 columns per wave (whole rows of the request),
// eight waves or two workgroups of four per CU: two waves per SIMD, so that one's VALU work runs beside the other's matrix
// instructions (four waves of 64 columns would read half as much from LDS, but past 256 registers every product's result
// has to come out of the accumulation file first: 1317 us where this form takes 992). K and V blocks of 64 keys go from the
// pages through registers into LDS (three K blocks, two V blocks), loaded two steps before they are stored (one in workgroups
// of four waves); one barrier per block. (Loads straight into LDS made the compiler wait for all of them before every LDS read.) V's layout in the cache is
// already the order in which it is read.
// Step n: the scores of block n + 1 (matrix core) under the exponentials of block n (VALU), then block n's products
// under the maxima of block n + 1. The rows of S^T's tiles hold the keys in the order in which P^T wants them (bits 2 and 3
// of the row exchanged), so weights never cross lanes. They are rounded to the cache's type for the product, as its values
// are, at most 2^8 above the reference maximum; scores, sums and products are float32.
// Measured, calls back to back: 4096 rows on 28,672 positions (16 / 8 heads of 128, fp16) 936 to 989 us by card, 1100 to 1040
// TFLOP/s: the card's power limit, at which a library product of 8192^3 reaches 1159; matrix cores busy 55 % of the cycles. A
// prompt of 2048 30 us (570 TFLOP/s): 4 us to start, 11 blocks of 1.9 us, 2 to store, 8 for the join.
template <typename T, int HD, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 1 : HD == 64 ? 3 : 2) void k_attn_tiles(AttnArgs a, uint32_t bytes) {
    using M = Mfma<T>;
    constexpr int KB = int(paged::kTileKeys), KS = HD / 16, DT = HD / 32, RB = HD * 2, BLK = KB * RB;
    constexpr int KR = RB + 16, KBLK = KB * KR;  // a K row in LDS is padded by 16 bytes: 16 rows lie in different banks
    constexpr int CH = RB / 16;            // 16-byte chunks of a K row
    constexpr int WK = KB / NW;            // keys of a block that a wave moves
    constexpr int LPB = WK * RB / 1024;    // its loads, of 1 KB each
    constexpr uint32_t GROUPS = paged::tile_groups(NW), COLS = paged::tile_cols(NW), SLOTS = paged::tile_slots(NW);
    // Workgroups that share a CU have one set of registers on the way to LDS (for heads of 64 three of them fit then, from
    // batches under way at once: 40 mixed requests 28.9 us against 31.1). Heads of 128 leave two of them room for two K
    // blocks: a block's place is free for the one after the next only when all waves have its scores, one more barrier a step.
    constexpr bool TIGHT = HD == 128 && NW == 4;
    constexpr int KN = TIGHT ? 2 : 3, SETS = NW == 4 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) uint8_t lds[KN * KBLK + 2 * BLK];  // K blocks n % KN, then V blocks n % 2
    uint32_t* const ends = reinterpret_cast<uint32_t*>(lds);                 // until the first block takes its place
    static_assert(sizeof(lds) >= 4 * paged::kMaxRequests);
    __shared__ uint32_t red[8];
    __shared__ uint32_t units_of_tile[64 * NW];
    __shared__ int chosen[3];
    __shared__ uint32_t arrived;
    __shared__ uint32_t odd;  // the first unit of the last piece that held values to take out
    const int t = threadIdx.x, lane = t & 63, wv = uniform(t >> 6), c32 = lane & 31, h = lane >> 5;
    const int group = int(a.qh / a.kvh), kvh = int(a.kvh), TR = int(COLS) / group;

    constexpr int kStart = int(paged::kTileStart);
    // ---- the units of every request, and this workgroup's
    // blocks of 64 keys of a request's first n tiles on one KV head: tile i's last row sees seen + min((i + 1) TR, rows) - 1
    // keys, at least one block. All full tiles but the clamped ones follow a slope. In even shares a tile weighs kStart units
    // more than it has, for its start.
    auto tile_keys = [&](const Request& q, int i) { return max(0, q.seen + min((i + 1) * TR, q.rows) - 1); };
    auto tile_units = [&](const Request& q, int i) { return max(1, (tile_keys(q, i) + KB - 1) / KB); };
    auto first_weight = [&](const Request& q, int n) {
        const int full = min(n, q.rows / TR);
        // tiles of one block: seen + (i + 1) TR - 1 <= 64
        const int ones = min(full, max(0, (KB + 1 - q.seen) / TR));
        uint32_t sum = uint32_t(ones);
        if (full > ones) sum += floor_sum64(uint32_t(full - ones), uint32_t(TR), uint32_t(q.seen + (ones + 1) * TR - 1 + KB - 1));
        if (n > full) sum += uint32_t(tile_units(q, full));
        return sum + uint32_t(n * kStart);
    };
    auto tiles_of = [&](const Request& q) { return (q.rows + TR - 1) / TR; };
    // ends[r] = the sum of f over the requests up to and with r
    auto scan_requests = [&](auto&& f) {
        const uint32_t per = (a.requests + 64 * NW - 1) / (64 * NW), r0 = min(t * per, a.requests), r1 = min(r0 + per, a.requests);
        uint32_t sum = 0;
        for (uint32_t r = r0; r < r1; ++r) {
            const Request q = request_of(a, r);
            sum = add_share(a, r, sum, q.rows > 0 ? f(q) : 0u);
            ends[r] = sum;
        }
        const uint32_t before = scan_sat(sum, red) - sum;
        for (uint32_t r = r0; r < r1; ++r) ends[r] += before;
        __syncthreads();
    };
    if (t == 0) odd = ~0u;
    Request rq{};
    auto enter = [&](int r) {
        rq = request_of(a, uint32_t(r));
        rq.row0 = uniform(rq.row0), rq.rows = uniform(rq.rows), rq.seen = uniform(rq.seen);
    };
    int r = 0, hk = 0, tile = 0, kfirst = 0;
    uint32_t u1 = 0, total = 0, G = 0, w = blockIdx.x;  // (weights of all items; not used where each has its own workgroups)
    uint32_t begin = 0;                                 // the weight before the item under way
    int parts = 0, mine = 0, lead = 0;                          // of an item with workgroups of its own
    // what the join has to know of a split item: written by the workgroup that begins it, by the others as none
    auto describe = [&](int parts, int base, int stride, int first, const Request& q, int row_first, int cols, int hk) {
        if (t != 0 || a.join_here) return;
        u32x4* d = reinterpret_cast<u32x4*>(a.ws + paged::kGroups) + 2 * w;
        d[0] = u32x4{uint32_t(parts), uint32_t(base), uint32_t(stride), uint32_t(first)};
        d[1] = u32x4{uint32_t(q.row0 + row_first), uint32_t(cols), uint32_t(hk), 0u};
    };
    auto describe_none = [&]() { describe(0, 0, 0, 0, Request{}, 0, 0, 0); };
    scan_requests([&](const Request& q) { return uint32_t(tiles_of(q)); });
    const uint32_t tiles_all = ends[a.requests - 1];
    if (tiles_all == 0 || tiles_all == kNoSum) {
        describe_none();
        return;
    }
    bool apart = uint64_t(tiles_all) * kvh <= GROUPS && tiles_all <= 256;
    uint32_t q = 0;
    if (apart) {
        // No more items than workgroups: each gets ceil(units / q) of its own, q the least that fits, so no workgroup starts
        // more than one piece (a start takes 4 us, the time of two units at head_dim 128). More parts than the square root of
        // half the longest item's units are not worth their join. All heads of a tile split alike; neighbouring workgroups,
        // which run on different XCDs, take different heads. Where whole workgroups fit the lengths badly, q far above the
        // mean, units shared out evenly are faster in spite of the second start: measured 171 us apart and 129 even at
        // q / mean = 1.85, 68 and 68 at 1.5, 88 and 94 at 1.67, 47 and 58 at 1.3.
        if (uint32_t(t) < tiles_all) {
            const int i = first_above(ends, int(a.requests), uint32_t(t));
            units_of_tile[t] = uint32_t(tile_units(request_of(a, uint32_t(i)), t - int(i ? ends[i - 1] : 0)));
        }
        __syncthreads();
        uint32_t n[4];
        const int held = int(tiles_all + 63) / 64;  // tiles of a lane
        float sum = 0.f, most = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            n[j] = uint32_t(lane + 64 * j) < tiles_all ? units_of_tile[lane + 64 * j] : 0u;
            sum += float(n[j]);
            most = fmaxf(most, float(n[j]));
        }
        const uint32_t room = GROUPS / uint32_t(kvh);
        uint32_t hi = uint32_t(uniform(int(wave_max(most)))), lo = uint32_t(uniform(int(wave_sum(sum)))) / room;
        const uint32_t even = lo;
        lo = min(max(max(lo, 1u), uint32_t(sqrtf(0.5f * float(hi)))), hi);
        while (lo < hi) {
            const uint32_t q = (lo + hi) >> 1;
            float need = 0.f;  // (a sum up to 2^24: exact; beyond, too many either way)
            const float by = 1.0f / float(q);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= held) continue;
                uint32_t c = uint32_t(float(n[j]) * by);  // n / q but for one (n is below 2^24 + 1)
                c += uint32_t(c * q < n[j]), c += uint32_t(c * q < n[j]), c -= uint32_t(c > 0 && (c - 1) * q >= n[j]);
                need += float(c);
            }
            if (uint32_t(uniform(int(wave_sum(need)))) <= room)
                hi = q;
            else
                lo = q + 1;
        }
        q = hi;
        apart = 4 * q <= 7 * even + 12;
    }
    if (apart) {
        const uint32_t own = uint32_t(t) < tiles_all ? (units_of_tile[t] + q - 1) / q : 0u, end = scan_sat(own, red);
        hk = int(w) % kvh;
        const uint32_t place = w / uint32_t(kvh);
        if (t == 0) chosen[0] = -1;
        __syncthreads();
        if (place < end && place >= end - own) chosen[0] = t, chosen[1] = int(own), chosen[2] = int(end - own);
        __syncthreads();
        const int at = uniform(chosen[0]);
        if (at < 0) {
            describe_none();
            return;
        }
        parts = uniform(chosen[1]), mine = int(place) - uniform(chosen[2]), lead = uniform(chosen[2]) * kvh + hk;
        r = uniform(first_above(ends, int(a.requests), uint32_t(at)));
        tile = at - uniform(r ? int(ends[r - 1]) : 0);
        enter(r);
    } else {
        __syncthreads();
        scan_requests([&](const Request& q) { return first_weight(q, tiles_of(q)) * uint32_t(kvh); });
        total = ends[a.requests - 1], G = min(uint32_t(gridDim.x), total);
        // workgroups of one XCD (every eighth) take neighbouring units, which share a KV head's blocks in its L2
        if (G == GROUPS) w = (blockIdx.x % 8) * (GROUPS / 8) + blockIdx.x / 8;
        if (w >= G) {
            describe_none();
            return;
        }
        const uint32_t u0 = uint32_t(uint64_t(total) * w / G);
        u1 = uint32_t(uint64_t(total) * (w + 1) / G);
        r = uniform(first_above(ends, int(a.requests), u0));
        enter(r);
        uint32_t in = u0 - (r ? uint32_t(uniform(int(ends[r - 1]))) : 0u);
        const int tiles = tiles_of(rq);
        const uint32_t per_head = uint32_t(uniform(int(first_weight(rq, tiles))));
        hk = int(in / per_head), in %= per_head;
        int lo = 0, hi = tiles - 1;  // the last tile whose first unit is at or before `in`
        while (lo < hi) {
            const int m = (lo + hi + 1) >> 1;
            if (first_weight(rq, m) <= in)
                lo = m;
            else
                hi = m - 1;
        }
        in = uint32_t(uniform(int(in - first_weight(rq, lo))));
        tile = uniform(lo), kfirst = max(0, int(in) - kStart), begin = u0 - in;
    }

    const __amdgpu_buffer_rsrc_t k_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.kc), 0, bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t v_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.vc), 0, bytes, 0x00020000);
    // this wave moves the WK keys of a block from WK wv on, 16 bytes per lane and load: both caches hold them in one piece
    int kst[LPB];  // where a K chunk goes in its block
#pragma unroll
    for (int i = 0; i < LPB; ++i) {
        const int p = 64 * i + lane, row = p / CH, ch = p % CH;  // row of the wave's WK, place in the row
        kst[i] = (WK * wv + row) * KR + ch * 16;
    }
    // operand reads: K row of matrix row c32 is key 16 (c32 / 16) + 8 (c32 / 4 % 2) + 4 (c32 / 8 % 2) + c32 % 4
    const int krow = (c32 & 19) | ((c32 & 4) << 1) | ((c32 & 8) >> 1);
    const int kbase = krow * KR + 16 * h, vbase = KN * KBLK + h * (8 * RB) + c32 * 16;

    constexpr int SW = int(paged::slot_words(COLS, HD));
    const __amdgpu_buffer_rsrc_t ws =
        __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, int(4 * (SLOTS + 2 * GROUPS * SW)), 0x00020000);
    bool described = false;

    for (;;) {
        // ---- a piece: blocks j0 .. j0 + nb - 1 of a tile
        const int units = tile_units(rq, tile), keys = tile_keys(rq, tile);
        const int j0 = apart ? int(uint64_t(uint32_t(units)) * mine / parts) : kfirst;
        const int nb = apart ? int(uint64_t(uint32_t(units)) * (mine + 1) / parts) - j0 : min(units, int(u1 - begin) - kStart) - j0;
        if (nb <= 0) break;  // (the start of an item, and none of its units)
        const int row_first = tile * TR, cols = min(TR, rq.rows - row_first) * group;
        const int cw = 32 * wv;  // this wave's first column
        // blocks that some column of the wave sees
        int nbw = 0;
        if (cw < cols) nbw = (max(0, rq.seen + row_first + min(cw + 31, cols - 1) / group) + KB - 1) / KB - j0;
        nbw = uniform(min(max(nbw, 0), nb));
        const int wave_seen = uniform(rq.seen + row_first + cw / group);  // keys that the wave's first column sees
        const int mycol = cw + c32, myrow = row_first + mycol / group, myhead = hk * group + mycol % group;
        const int vis = rq.seen + myrow;  // keys that this lane's column sees
        u32x4 qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = u32x4{0u, 0u, 0u, 0u};
            if (mycol < cols)
                qf[s] = *reinterpret_cast<const u32x4*>(
                    static_cast<const T*>(a.q) + (size_t(rq.row0 + myrow) * a.qh + myhead) * HD + 16 * s + 8 * h);
        }
        const uint32_t* const trow = a.table + size_t(r) * a.blocks;
        // the pages of 16 blocks at a time, lane 4 i + p those of part p (16 keys) of block i: its place in the caches for
        // this wave's part is a lane read, the set of parts without a page four bits of a ballot
        auto page_ids = [&](int j) __attribute__((always_inline)) {
            return trow[min(uint32_t((j0 + j) * KB + 16 * lane) >> a.page_log2, a.blocks - 1)];
        };
        uint32_t ids = page_ids(0), ids_next = ids;
        uint64_t no_page = __ballot(ids >= a.pages);
        auto locate = [&](int j, int& soff, uint32_t& bad) __attribute__((always_inline)) {
            if ((j & 15) == 8) ids_next = page_ids((j & ~15) + 16);
            if ((j & 15) == 0 && j) {
                ids = ids_next;
                no_page = __ballot(ids >= a.pages);
            }
            bad = uint32_t(no_page >> (4 * (j & 15))) & 15u;
            const uint32_t id = uint32_t(__builtin_amdgcn_readlane(int(ids), 4 * (j & 15) + (WK * wv >> 4)));
            const uint32_t off = uint32_t((j0 + j) * KB + WK * wv) & ((1u << a.page_log2) - 1);
            soff = id < a.pages ? int((((id * uint32_t(kvh) + hk) << a.page_log2) + off) * RB) : 0;
        };
        // the chunks of this wave on their way to LDS: SETS blocks of each cache
        u32x4 rk[SETS][LPB], rv[SETS][LPB];
        auto load_k = [&](auto set, int i, int soff) __attribute__((always_inline)) {
            rk[decltype(set)::value % SETS][i] = __builtin_amdgcn_raw_buffer_load_b128(k_rsrc, 16 * lane + 1024 * i, soff, 0);
        };
        auto load_v = [&](auto set, int i, int soff) __attribute__((always_inline)) {
            rv[decltype(set)::value % SETS][i] = __builtin_amdgcn_raw_buffer_load_b128(v_rsrc, 16 * lane + 1024 * i, soff, 0);
        };
        auto store_k = [&](auto set, int i, int slot) __attribute__((always_inline)) {
            *reinterpret_cast<u32x4*>(lds + slot * KBLK + kst[i]) = rk[decltype(set)::value % SETS][i];
        };
        auto store_v = [&](auto set, int i, int slot) __attribute__((always_inline)) {
            *reinterpret_cast<u32x4*>(lds + KN * KBLK + slot * BLK + 1024 * (LPB * wv + i) + 16 * lane) =
                rv[decltype(set)::value % SETS][i];
        };
        const int tile_seen = rq.seen + row_first;  // keys that the tile's first row sees: all of its columns do
        auto hide_v = [&](auto set, int j, uint32_t bad) __attribute__((always_inline)) {
            const int left = keys - (j0 + j) * KB;  // keys of the block that any column sees
            if (left < KB || bad) {  // uniform: what is hidden may be anything, and zero times NaN is NaN
#pragma unroll
                for (int i = 0; i < LPB; ++i) {
                    const int in = (bad >> (WK * wv >> 4) & 1u) ? 0 : left - WK * wv - i * 1024 / (8 * RB) * 8;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        rv[decltype(set)::value % SETS][i][e] &= (2 * e < in ? 0x0000FFFFu : 0u) | (2 * e + 1 < in ? 0xFFFF0000u : 0u);
                }
            }
            if ((j0 + j + 1) * KB > tile_seen) {
                bool any = false;
#pragma unroll
                for (int i = 0; i < LPB; ++i) any |= take_odd<T>(rv[decltype(set)::value % SETS][i]);
                if (any) odd = begin;
            }
        };
        f32x16 sa, sb, o[DT];  // scores of a block's first and last 32 keys; products, [dim tile]
        float m_run = -INFINITY, mc = 0.f, l_run = 0.f;  // reference maximum, the same in the exponent (0: none yet), sum
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
        auto join_halves = [&](float m) __attribute__((always_inline)) {  // the maximum over lanes l and l + 32
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
            return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
        };
        auto maximum = [&](f32x16& s) __attribute__((always_inline)) {
            float m = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) m = fmaxf(m, s[e]);
            return join_halves(m);
        };
        // the reference maximum moves where a column leaves it behind by more than 8 in the exponent
        auto follow = [&](float mx) __attribute__((always_inline)) {
            const bool grow = (mx - m_run) * a.scale_log2 > 8.0f;  // false for NaN (both -inf)
            if (__any(grow)) {
                const float alpha = grow ? __builtin_amdgcn_exp2f((m_run - mx) * a.scale_log2) : 1.0f;
                m_run = grow ? mx : m_run;
                mc = m_run == -INFINITY ? 0.f : m_run * a.scale_log2 - kUp<T>;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= alpha;
            }
        };
        // hides what the columns do not see of the 32 keys first
        auto settle = [&](int j, int kt, uint32_t bad, f32x16& s, float mx) __attribute__((always_inline)) {
            const int kb = (j0 + j) * KB + 32 * kt;
            if (j >= nbw) {  // behind the last block: nothing to see
                mx = -INFINITY;
            } else if (kb + 32 > wave_seen || bad) {  // uniform
                const int lim = vis - kb - 8 * h;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (16 * (e >> 3) + (e & 7) >= lim || (bad >> (2 * kt + (e >> 3)) & 1u)) s[e] = -INFINITY;
                mx = maximum(s);
            }
            follow(mx);
        };
        // 32 keys: the scores of the next 32 (matrix core) under the weights of these (VALU), then their products under the
        // last of the weights and the next ones' maxima, each operand read two instructions ahead.
        u32x4 kp[2];  // the first two operands of the next scores, read under the products before them
        auto half = [&](int kslot, int nkt, f32x16& nxt, int vslot, int kt, f32x16& cur, int pslot, int pkt,
                        auto&& side) __attribute__((always_inline)) {
            const uint8_t* k0 = lds + kslot * KBLK + nkt * 32 * KR + kbase;
            const uint8_t* p0 = lds + pslot * KBLK + pkt * 32 * KR + kbase;
            const uint8_t* v0 = lds + vslot * BLK + vbase + kt * 32 * RB;
            auto read_k = [&](int s) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4*>(k0 + 32 * s); };
            auto read_v = [&](int i) __attribute__((always_inline)) {
                return *reinterpret_cast<const u32x4*>(v0 + (i / DT) * 16 * RB + (i % DT) * 512);
            };
            constexpr int NV = 2 * DT;
            u32x4 kf[KS], vf[NV], pb[2];  // (pb: weights packed as the products' operands, [16 keys])
            // two weights: pair p of 8
            auto weigh = [&](int p) __attribute__((always_inline)) {
                const float x = __builtin_amdgcn_exp2f(fmaf(cur[2 * p], a.scale_log2, -mc));
                const float y = __builtin_amdgcn_exp2f(fmaf(cur[2 * p + 1], a.scale_log2, -mc));
                l_run += x;
                l_run += y;
                pb[p / 4][p % 4] = pack<T>(x, y);
                asm volatile("" : "+v"(l_run));  // (the sums stay here)
            };
            constexpr int EARLY = 6;  // pairs under the scores; the other two under the first products
#pragma unroll
            for (int e = 0; e < 16; ++e) nxt[e] = 0.f;
            kf[0] = kp[0], kf[1] = kp[1];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s + 2 < KS) kf[s + 2] = read_k(s + 2);
                if (s + 2 >= KS) vf[s + 2 - KS] = read_v(s + 2 - KS);
                side(s, KS + NV);
                nxt = M::m32(kf[s], qf[s], nxt);
#pragma unroll
                for (int p = EARLY * s / KS; p < EARLY * (s + 1) / KS; ++p) weigh(p);
            }
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (i + 2 < NV) vf[i + 2] = read_v(i + 2);
                if (i + 2 >= NV) kp[i + 2 - NV] = *reinterpret_cast<const u32x4*>(p0 + 32 * (i + 2 - NV));
                side(KS + i, KS + NV);
                o[i % DT] = M::m32(vf[i], pb[i / DT], o[i % DT]);
                if (i < DT)
#pragma unroll
                    for (int p = EARLY + 2 * i / DT; p < EARLY + 2 * (i + 1) / DT; ++p) weigh(p);
#pragma unroll
                for (int p = i < 2 ? 0 : 8 * (i - 2) / (NV - 2); i >= 2 && p < 8 * (i - 1) / (NV - 2); ++p)
                    m = fmaxf(fmaxf(m, nxt[2 * p]), nxt[2 * p + 1]);  // (the last scores are two products old)
            }
            return join_halves(m);
        };

        // Step n stores K(n + 2) and V(n + 1) under its second half, loaded by step n - 2 (a block that is not in the XCD's L2
        // takes about a step to arrive), and loads K(n + 4) and V(n + 3) into the registers that this frees (behind the last
        // block: the last one again, never read). With one set of registers: loaded by step n - 1, and K(n + 3) and V(n + 2).
        using A0 = std::integral_constant<int, 0>;
        using A1 = std::integral_constant<int, 1>;
        int s1, s2, s3, s4;
        uint32_t b0, b1, b2, b3, b4;
        locate(0, s1, b0);
#pragma unroll
        for (int i = 0; i < LPB; ++i) load_k(A0{}, i, s1), load_v(A0{}, i, s1);
        locate(min(1, nb - 1), s1, b1);
        if constexpr (SETS == 2)
#pragma unroll
            for (int i = 0; i < LPB; ++i) load_k(A1{}, i, s1);
        locate(min(2, nb - 1), s2, b2);
        locate(min(3, nb - 1), s3, b3);
        lds_barrier();  // the blocks of the piece before this one are read
        hide_v(A0{}, 0, b0);
#pragma unroll
        for (int i = 0; i < LPB; ++i) {
            store_k(A0{}, i, 0);
            load_k(A0{}, i, SETS == 2 ? s2 : s1);
            store_v(A0{}, i, 0);
            load_v(A0{}, i, s1);
        }
#pragma unroll
        for (int i = 0; i < LPB; ++i) {
            store_k(A1{}, i, 1);
            load_k(A1{}, i, SETS == 2 ? s3 : s2);
            if constexpr (SETS == 2) load_v(A1{}, i, s2);
        }
        s4 = s3, b4 = b3;
        lds_barrier();
        if (nbw > 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sa[e] = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) sa = M::m32(*reinterpret_cast<const u32x4*>(lds + kbase + 32 * s), qf[s], sa);
            settle(0, 0, b0, sa, maximum(sa));
#pragma unroll
            for (int i = 0; i < 2; ++i) kp[i] = *reinterpret_cast<const u32x4*>(lds + 32 * KR + kbase + 32 * i);
        }
        int kslot = 0, n = 0;  // kslot = n % KN
        auto none = [](int, int) {};
        // PLAIN: every column sees all of this block and the next, all have pages, and more follow: nothing to ask
        auto step = [&](auto set, auto plain) __attribute__((always_inline)) {
            constexpr bool PLAIN = decltype(plain)::value;
            const int kslot1 = kslot == KN - 1 ? 0 : kslot + 1, kslot2 = kslot1 == KN - 1 ? 0 : kslot1 + 1, vslot = n & 1;
            if (n) lds_barrier();
            if (PLAIN || n + 4 < nb) locate(n + 4, s4, b4);
            if (!PLAIN && n + 1 < nb) hide_v(set, n + 1, b1);
            // one store or load of a chunk: 4 LPB of them shared out over the parts of a half
            auto moves = [&](int part, int parts) __attribute__((always_inline)) {
#pragma unroll
                for (int x = 4 * LPB * part / parts; x < 4 * LPB * (part + 1) / parts; ++x) {
                    const int i = x >> 2;
                    if ((x & 3) == 0) store_k(set, i, kslot2);
                    if ((x & 3) == 1) load_k(set, i, SETS == 2 ? s4 : s3);
                    if ((x & 3) == 2) store_v(set, i, 1 - vslot);
                    if ((x & 3) == 3) load_v(set, i, SETS == 2 ? s3 : s2);
                }
            };
            const bool act = PLAIN ? nbw > 0 : n < nbw;
            auto first_half = [&]() __attribute__((always_inline)) {
                const float mx = half(kslot, 1, sb, vslot, 0, sa, kslot1, 0, none);
                if constexpr (PLAIN)
                    follow(mx);
                else
                    settle(n, 1, b0, sb, mx);
            };
            auto second_half = [&]() __attribute__((always_inline)) {
                const float mx = half(kslot1, 0, sa, vslot, 1, sb, kslot1, 1, moves);  // (scores behind the last block: not used)
                if constexpr (PLAIN)
                    follow(mx);
                else
                    settle(n + 1, 0, b1, sa, mx);
            };
            if constexpr (TIGHT) {
                if (act) first_half();
                lds_barrier();
                if (act)
                    second_half();
                else
                    moves(0, 1);
            } else if (act) {
                first_half();
                second_half();
            } else {
                moves(0, 1);
            }
            s2 = s3, s3 = s4, b0 = b1, b1 = b2, b2 = b3, b3 = b4, kslot = kslot1, ++n;
        };
        const int plain = (b0 | b1 | b2 | b3) || no_page ? 0 : min(nb - 4, (rq.seen + row_first) / KB - 1 - j0);
        while (n + 1 < plain && !no_page) {  // (no_page: among the 16 blocks from n + 3 on)
            step(A0{}, std::true_type{});
            step(A1{}, std::true_type{});
        }
        for (;;) {
            step(A0{}, std::false_type{});
            if (n >= nb) break;
            step(A1{}, std::false_type{});
            if (n >= nb) break;
        }
        {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
            l_run = __uint_as_float(x[0]) + __uint_as_float(x[1]);
        }

        if (uint32_t(uniform(int(odd))) == begin) {  // adds the values that hide_v has taken out, from the cache once more
            const int end = min((j0 + nb) * KB, keys);
#pragma unroll 1
            for (int k = max(j0 * KB, tile_seen / KB * KB); k < end; k += 16) {
                const uint32_t id = uint32_t(uniform(int(trow[min(uint32_t(k) >> a.page_log2, a.blocks - 1)])));
                if (id >= a.pages) continue;
                const int soff = int((((id * uint32_t(kvh) + hk) << a.page_log2) + (uint32_t(k) & ((1u << a.page_log2) - 1))) * RB);
                const int lim = vis - k - 8 * h;
                u32x4 sees;
#pragma unroll
                for (int e = 0; e < 4; ++e) sees[e] = pack<T>(2 * e < lim ? 1.f : 0.f, 2 * e + 1 < lim ? 1.f : 0.f);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    f32x16 counts;
#pragma unroll
                    for (int e = 0; e < 16; ++e) counts[e] = 0.f;
                    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(v_rsrc, 8 * RB * h + 512 * d + 16 * c32, soff, 0);
                    counts = M::m32(odd_codes<T>(x), sees, counts);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] = add_odd(o[d][e], counts[e]);
                    __builtin_amdgcn_sched_barrier(0);  // (one tile of counts at a time)
                }
            }
        }

        auto write = [&]() __attribute__((always_inline)) {
            const float inv = l_run != 0.f ? 1.0f / l_run : 0.f;  // no key at all: zeros
            T* y = static_cast<T*>(a.y) + (size_t(rq.row0 + myrow) * a.qh + myhead) * HD + 4 * h;
            if (mycol < cols) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e)  // dims 32 d + 8 e + 4 h ..
                        *reinterpret_cast<uint2*>(y + 32 * d + 8 * e) =
                            make_uint2(pack_mean<T>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv),
                                       pack_mean<T>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv));
            }
        };
        // the item's parts: part i in slot base + i stride (+ 1 for the first, which its workgroup begins)
        int base = 2 * lead, stride = 2 * kvh, first = 0;
        if (!apart) {
            const uint32_t unit0 = begin + uint32_t(kStart);
            auto group_of = [&](uint32_t x) { return int(((uint64_t(x) + 1) * G - 1) / total); };
            lead = group_of(unit0), parts = group_of(unit0 + uint32_t(units) - 1) - lead + 1, mine = int(w) - lead;
            base = 2 * lead, stride = 2, first = 1;
        }
        if (parts == 1) {
            write();
        } else {
            if (mine == 0) {
                describe(parts, base, stride, first, rq, row_first, cols, hk);
                described = true;
            }
            if (cw < cols) {  // 16 bytes i of lane l: (4 DT wave + i) 64 + l, after the maxima and sums
                const int slot = int(SLOTS) + (base + mine * stride + (mine ? 0 : first)) * SW;
                if (h == 0) store_part2(ws, slot + 2 * mycol, m_run, l_run);
#pragma unroll
                for (int i = 0; i < 4 * DT; ++i) {
                    const f32x16& x = o[i >> 2];
                    const int e = 4 * (i & 3);
                    store_part(ws, slot + 2 * int(COLS) + ((wv * 4 * DT + i) * 64 + lane) * 4,
                               f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]});
                }
            }
            if (a.join_here) {
                __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0): this wave's stores are performed
                lds_barrier();
                uint32_t* const counter = a.ws + lead;
                if (t == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                lds_barrier();
                if (uint32_t(uniform(int(arrived))) == uint32_t(parts - 1)) {
                    if (cw < cols)
#pragma unroll 1
                        for (int d = 0; d < 4; ++d)
                            join_item<T, HD, NW, kDeviceScope>(
                                a, Split{parts, base, stride, first, rq.row0 + row_first, cols, hk}, wv, d, lane);
                    if (t == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
        if (apart) break;
        // ---- the next piece
        begin += uint32_t(kStart + units);
        kfirst = 0;
        if (begin + uint32_t(kStart) >= u1) break;
        if (++tile >= tiles_of(rq)) {
            tile = 0;
            if (++hk >= kvh) {
                hk = 0;
                do
                    enter(++r);
                while (rq.rows < 1 && r < int(a.requests) - 1);
            }
        }
    }
    if (!described) describe_none();
}

// The joins of k_attn_tiles' split items where they may have many parts, a launch of its own for all CUs (kJoinHere). Block
// (item, wave of the tile): its four waves take a quarter of each column's dims each.
template <typename T, int HD, int NW>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    const int lead = blockIdx.x / NW, wv = blockIdx.x % NW, t = threadIdx.x;
    const u32x4* d = reinterpret_cast<const u32x4*>(a.ws + paged::kGroups) + 2 * lead;
    const u32x4 d0 = d[0], d1 = d[1];
    const Split p{uniform(int(d0[0])), uniform(int(d0[1])), uniform(int(d0[2])), uniform(int(d0[3])), int(d1[0]), int(d1[1]), int(d1[2])};
    if (p.parts == 0 || 32 * wv >= p.cols) return;
    join_item<T, HD, NW, 0>(a, p, wv, t >> 6, t & 63);
}

}  // namespace

// ---------------------------------------------------------------- launchers

static uint32_t log2_of(uint32_t page) { return uint32_t(__builtin_ctz(page)); }
static float f32_of(uint32_t b) {
    float f;
    std::memcpy(&f, &b, 4);
    return f;
}
static uint32_t dtype_of(const PreparedDispatch& pd, int field) {
    for (const TokenUse& u : pd.tokens)
        if (u.field == field) return u.row.dtype();
    return 0;
}

// rows and new pages are shared out over at most 512 workgroups
static uint32_t plan_blocks(uint32_t tokens) { return std::min(512u, (tokens + 255) / 256); }

// past, fresh, free, table, starts, context, positions, slots, counts, requests, blocks, page, pages, free_count, tokens
static void l_plan(const PreparedDispatch& pd, void* const* p, hipStream_t s) {
    const uint32_t* w = pd.words.data();
    auto u = [&](int i) { return (uint32_t*)p[i]; };
    hipLaunchKernelGGL(k_paged_plan, dim3(plan_blocks(w[15])), dim3(256), 0, s, u(0), u(1), u(2), u(3), u(4), u(5), u(6),
                       u(7), u(8), w[10], w[11], log2_of(w[12]), w[13], w[14], w[15]);
}

// qkv, q_norm, k_norm, cos_table, sin_table, starts, positions, slots, q, k_cache, v_cache, requests, tokens, q_heads,
// kv_heads, head_dim, max_pos, page, pages, eps
// The grid of 48: waves of queries and keys, then waves of values. A wave takes 1024 elements of a row's query and key heads,
// or, from 4096 rows on, all of them, so that the row's rotation is loaded once (2048 rows: 8.8 us in parts, 9.9 whole; 4096:
// 15.8 and 16.0; 9,200 rows of 40 heads in bf16 49.4 and 47.0, of 24 in float32 46.1 and 48.4); 8 rows x 128 elements of the
// value heads.
struct AppendGrid {
    uint32_t parts, qk_blocks, v_chunks, v_blocks;
};
static AppendGrid append_grid(const uint32_t* w) {
    const uint64_t T = w[13];
    AppendGrid g;
    g.parts = T >= 4096 ? 1 : uint32_t(((uint64_t(w[14]) + w[15]) * w[16] + 1023) / 1024);
    g.qk_blocks = uint32_t((T * g.parts + 3) / 4);
    g.v_chunks = uint32_t((uint64_t(w[15]) * w[16] + 127) / 128);
    g.v_blocks = uint32_t(((T + 7) / 8 * g.v_chunks + 3) / 4);
    return g;
}
template <typename IN, typename T, int HD>
static void launch_append(const uint32_t* w, const Physical& d, void* const* p, hipStream_t s) {
    const AppendGrid g = append_grid(w);
    hipLaunchKernelGGL((k_paged_append<IN, T, HD>), dim3(d.x, d.y), dim3(256), 0, s,
                       (const IN*)p[0], (const uint16_t*)p[1], (const uint16_t*)p[2], (const float*)p[3],
                       (const float*)p[4], (const uint32_t*)p[5], (const uint32_t*)p[6], (const uint32_t*)p[7], (T*)p[8],
                       (T*)p[9], (T*)p[10], w[12], w[13], w[14], w[15], w[17], log2_of(w[18]), w[19], f32_of(w[20]),
                       g.qk_blocks, g.parts, g.v_chunks);
}
template <typename IN, typename T>
static void launch_append(const uint32_t* w, const Physical& d, void* const* p, hipStream_t s) {
    if (w[16] == 64)
        launch_append<IN, T, 64>(w, d, p, s);
    else
        launch_append<IN, T, 128>(w, d, p, s);
}
static void l_append(const PreparedDispatch& pd, void* const* p, hipStream_t s) {
    const uint32_t* w = pd.words.data();
    const bool half = dtype_of(pd, 8) == F16;
    if (dtype_of(pd, 0) == F32) {
        if (half)
            launch_append<float, _Float16>(w, pd.physical, p, s);
        else
            launch_append<float, __bf16>(w, pd.physical, p, s);
    } else if (half) {
        launch_append<_Float16, _Float16>(w, pd.physical, p, s);
    } else {
        launch_append<__bf16, __bf16>(w, pd.physical, p, s);
    }
}

// q, k_cache, v_cache, table, starts, context, y, workspace, requests, tokens, max_fresh, q_heads, kv_heads, head_dim,
// blocks, page, pages, scale
// the most new rows of a request in the dispatch, and whether every item's columns fit the kernel for few
static uint32_t most_fresh(const uint32_t* w) { return w[11] ? std::min(w[11], w[10]) : w[10]; }
// (the kernel for few against the tiles at 16 columns: 16 requests of 4 rows on 2000 positions 23 us and 32, 64 of one row 86
// and 101; past 16 a second tile of columns would double its registers)
static bool few_columns(const uint32_t* w) {
    return w[13] && uint64_t(most_fresh(w)) * (w[12] / w[13]) <= paged::kRowsCols;
}
static uint32_t tile_waves_of(const uint32_t* w) { return paged::tile_waves(w[9], w[10], w[14], w[13] ? w[12] / w[13] : 0); }
template <typename T, int HD, int NW>
static void launch_tiles(const AttnArgs& a, uint32_t bytes, hipStream_t s) {
    constexpr uint32_t groups = paged::tile_groups(NW);
    hipLaunchKernelGGL((k_attn_tiles<T, HD, NW>), dim3(groups), dim3(64 * NW), 0, s, a, bytes);
    if (!a.join_here) hipLaunchKernelGGL((k_attn_join<T, HD, NW>), dim3(groups * NW), dim3(256), 0, s, a);
}
template <typename T, int HD>
static void launch_attn(const uint32_t* w, void* const* p, hipStream_t s) {
    const float scale_log2 = f32_of(w[18]) * 1.4426950408889634f;
    const AttnArgs a{p[0], p[1], p[2], (const uint32_t*)p[3], (const uint32_t*)p[4], (const uint32_t*)p[5], p[6],
                     (uint32_t*)p[7], w[9], w[10], most_fresh(w), w[12], w[13], w[15], log2_of(w[16]), w[17], uint32_t(uint64_t(w[15]) * w[16] <= paged::kJoinHere),
                     scale_log2};
    const uint32_t bytes = uint32_t(uint64_t(w[17]) * w[16] * w[13] * HD * 2);  // of each cache
    if (few_columns(w))
        hipLaunchKernelGGL((k_attn_rows<T, HD>), dim3(paged::kRowsGroups), dim3(256), 0, s, a, bytes, bytes);
    else if (tile_waves_of(w) == 8)
        launch_tiles<T, HD, 8>(a, bytes, s);
    else
        launch_tiles<T, HD, 4>(a, bytes, s);
}
static void l_attn(const PreparedDispatch& pd, void* const* p, hipStream_t s) {
    const uint32_t* w = pd.words.data();
    const bool half = dtype_of(pd, 0) == F16;
    if (w[14] == 64) {
        if (half)
            launch_attn<_Float16, 64>(w, p, s);
        else
            launch_attn<__bf16, 64>(w, p, s);
    } else if (half) {
        launch_attn<_Float16, 128>(w, p, s);
    } else {
        launch_attn<__bf16, 128>(w, p, s);
    }
}

const LaunchFn* paged_launchers() {
    static const LaunchFn t[] = {l_plan, l_append, l_attn};
    return t;
}

// ---------------------------------------------------------------- catalog entries (ids 47..49)

#define DT(x) (1u << (x))
#define TOK_R(n, m) FieldSpec{n, FieldKind::Token, Access::Read, m, nullptr}
#define TOK_W(n, m) FieldSpec{n, FieldKind::Token, Access::Write, m, nullptr}
#define TOK_RW(n, m) FieldSpec{n, FieldKind::Token, Access::ReadWrite, m, nullptr}
#define U32F(n) FieldSpec{n, FieldKind::U32, Access::None, 0, nullptr}
#define F32F(n) FieldSpec{n, FieldKind::F32, Access::None, 0, nullptr}

static void need(const uint32_t* counts, int field, uint64_t elems, const char* kernel, const char* what) {
    if (counts[field] < elems)
        contract_fail("%s.%s holds %u elements; the dispatch touches %llu", kernel, what, counts[field],
                      (unsigned long long)elems);
}
// a product of three words (each below 2^32, the last two of them dimensions of a tensor row) that cannot wrap
static uint64_t times(uint64_t a, uint64_t b, uint64_t c = 1) {
    const __uint128_t v = (__uint128_t)a * b * c;
    return v >> 64 ? ~0ull : uint64_t(v);
}

static void need_step(const char* n, uint32_t requests, uint32_t tokens) {
    if (requests < 1 || requests > paged::kMaxRequests)
        contract_fail("%s: requests must be in 1 .. %u", n, paged::kMaxRequests);
    if (tokens < 1) contract_fail("%s: tokens must be at least 1", n);
}
static void need_pages(const char* n, uint32_t page, uint32_t pages) {
    if (!paged::page_ok(page)) contract_fail("%s: page must be a power of two in 16 .. 256", n);
    if (pages < 1 || times(pages, page) > 0xFFFFFFFFull)
        contract_fail("%s: pages must be at least 1, and pages * page at most 2^32 - 1", n);
}
static void need_table(const char* n, uint32_t blocks, uint32_t page) {
    if (blocks < 1 || times(blocks, page) > 1ull << 30)
        contract_fail("%s: blocks must be at least 1, and blocks * page at most 2^30", n);
}
static void need_heads(const char* n, uint32_t qh, uint32_t kvh, uint32_t hd) {
    if (kvh < 1 || qh < 1 || qh % kvh) contract_fail("%s: kv_heads must divide q_heads", n);
    if (hd != 64 && hd != 128) contract_fail("%s: head_dim must be 64 or 128", n);
}
static void same_dtype(const char* n, const std::vector<TokenUse>& tokens, std::initializer_list<int> fields) {
    uint32_t first = 0;
    for (const TokenUse& u : tokens)
        for (int f : fields)
            if (u.field == f) {
                if (!first) first = u.row.dtype();
                if (u.row.dtype() != first)
                    contract_fail("%s: %s and %s cannot be mixed in one dispatch", n, dtype_name(first),
                                  dtype_name(u.row.dtype()));
            }
}

std::vector<KernelSpec> paged_catalog() {
    std::vector<KernelSpec> c;
    const uint32_t U = DT(U32), H = DT(F16) | DT(BF16);
    // 47 paged_plan
    c.push_back({"paged_plan", "paged", {256, 1, 1}, true,
                 [](const uint32_t* w) { return Grid3{plan_blocks(w[15]), 1, 1}; },
                 {TOK_R("past", U), TOK_R("fresh", U), TOK_R("free", U), TOK_RW("table", U), TOK_W("starts", U),
                  TOK_W("context", U), TOK_W("positions", U), TOK_W("slots", U), TOK_W("counts", U), U32F("requests"),
                  U32F("blocks"), U32F("page"), U32F("pages"), U32F("free_count"), U32F("tokens")},
                 [](const uint32_t* w, const uint32_t* c) {
                     const char* n = "paged_plan";
                     const uint32_t R = w[10], blocks = w[11], page = w[12], pages = w[13], free_count = w[14], T = w[15];
                     need_step(n, R, T);
                     need_pages(n, page, pages);
                     need_table(n, blocks, page);
                     need(c, 0, R, n, "past");
                     need(c, 1, R, n, "fresh");
                     need(c, 2, free_count, n, "free");
                     need(c, 3, times(R, blocks), n, "table");
                     need(c, 4, uint64_t(R) + 1, n, "starts");
                     need(c, 5, R, n, "context");
                     need(c, 6, T, n, "positions");
                     need(c, 7, T, n, "slots");
                     need(c, 8, 3, n, "counts");
                 }});
    // 48 qk_norm_rope_append_paged
    c.push_back({"qk_norm_rope_append_paged", "paged", {256, 1, 1}, true,
                 [](const uint32_t* w) {
                     const AppendGrid g = append_grid(w);
                     return Grid3{int64_t(g.qk_blocks) + g.v_blocks, 1, 1};
                 },
                 {TOK_R("qkv", H | DT(F32)), TOK_R("q_norm", DT(BF16)), TOK_R("k_norm", DT(BF16)),
                  TOK_R("cos_table", DT(F32)), TOK_R("sin_table", DT(F32)), TOK_R("starts", U), TOK_R("positions", U),
                  TOK_R("slots", U), TOK_W("q", H), TOK_RW("k_cache", H), TOK_RW("v_cache", H), U32F("requests"),
                  U32F("tokens"), U32F("q_heads"), U32F("kv_heads"), U32F("head_dim"), U32F("max_pos"), U32F("page"),
                  U32F("pages"), F32F("eps")},
                 [](const uint32_t* w, const uint32_t* c) {
                     const char* n = "qk_norm_rope_append_paged";
                     const uint32_t R = w[12], T = w[13], qh = w[14], kvh = w[15], hd = w[16], mp = w[17], page = w[18],
                                    pages = w[19];
                     need_step(n, R, T);
                     need_heads(n, qh, kvh, hd);
                     need_pages(n, page, pages);
                     if (mp < 1) contract_fail("%s: max_pos must be at least 1", n);
                     need(c, 0, times(T, uint64_t(qh) + 2 * uint64_t(kvh), hd), n, "qkv");
                     need(c, 1, hd, n, "q_norm");
                     need(c, 2, hd, n, "k_norm");
                     need(c, 3, times(mp, hd / 2), n, "cos_table");
                     need(c, 4, times(mp, hd / 2), n, "sin_table");
                     need(c, 5, uint64_t(R) + 1, n, "starts");
                     need(c, 6, T, n, "positions");
                     need(c, 7, T, n, "slots");
                     need(c, 8, times(T, qh, hd), n, "q");
                     need(c, 9, times(uint64_t(pages) * page, kvh, hd), n, "k_cache");
                     need(c, 10, times(uint64_t(pages) * page, kvh, hd), n, "v_cache");
                 },
                 [](const std::vector<TokenUse>& t) {
                     same_dtype("qk_norm_rope_append_paged", t, {8, 9, 10});
                     if (t[0].row.dtype() != F32) same_dtype("qk_norm_rope_append_paged", t, {0, 8});
                 }});
    // 49 attention_paged (the catalog's thread count is that of the kernel for few columns; the tiles' have 256 or 512, and a
    // second launch may join their split items)
    c.push_back({"attention_paged", "paged", {256, 1, 1}, false,
                 [](const uint32_t* w) {
                     return Grid3{int64_t(few_columns(w) ? paged::kRowsGroups : paged::tile_groups(tile_waves_of(w))), 1, 1};
                 },
                 {TOK_R("q", H), TOK_R("k_cache", H), TOK_R("v_cache", H), TOK_R("table", U), TOK_R("starts", U),
                  TOK_R("context", U), TOK_W("y", H), TOK_RW("workspace", U), U32F("requests"), U32F("tokens"),
                  U32F("max_fresh"), U32F("q_heads"), U32F("kv_heads"), U32F("head_dim"), U32F("blocks"), U32F("page"),
                  U32F("pages"), F32F("scale")},
                 [](const uint32_t* w, const uint32_t* c) {
                     const char* n = "attention_paged";
                     const uint32_t R = w[9], T = w[10], qh = w[12], kvh = w[13], hd = w[14], blocks = w[15], page = w[16],
                                    pages = w[17];
                     need_step(n, R, T);
                     need_heads(n, qh, kvh, hd);
                     need_pages(n, page, pages);
                     need_table(n, blocks, page);
                     const float scale = f32_of(w[18]);
                     if (!(scale > 0.f) || std::isinf(scale)) contract_fail("%s: scale must be positive and finite", n);
                     if (qh / kvh > paged::kMaxTileCols)
                         contract_fail("%s: at most %u query heads per KV head", n, paged::kMaxTileCols);
                     // units: a tile of a request's rows (at least one a request) x the blocks of keys, on every KV head
                     const uint64_t tiles = R + uint64_t(T) / (paged::tile_cols(tile_waves_of(w)) / (qh / kvh));
                     if (times(few_columns(w) ? R : tiles, kvh,
                               uint64_t(blocks) * page / paged::kTileKeys + 1 + paged::kTileStart) > 1ull << 31)
                         contract_fail("%s: rows * kv_heads * blocks * page are more than one dispatch shares out", n);
                     need(c, 0, times(T, qh, hd), n, "q");
                     need(c, 1, times(uint64_t(pages) * page, kvh, hd), n, "k_cache");
                     need(c, 2, times(uint64_t(pages) * page, kvh, hd), n, "v_cache");
                     need(c, 3, times(R, blocks), n, "table");
                     need(c, 4, uint64_t(R) + 1, n, "starts");
                     need(c, 5, R, n, "context");
                     need(c, 6, times(T, qh, hd), n, "y");
                     need(c, 7, paged::workspace_words(R, T, qh, kvh, hd), n, "workspace");
                 },
                 [](const std::vector<TokenUse>& t) { same_dtype("attention_paged", t, {0, 1, 2, 6}); }});
    return c;
}

}  // namespace lrm
