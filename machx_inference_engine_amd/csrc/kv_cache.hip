// kv_cache.hip — rotary positions and the paged key-value cache: rotation of query and key rows, writing (with Q8_0 quantisation) and reading back.
#include <math.h>

#include "mxq_device.h"
#include "mxq_host.h"

namespace mxq {

constexpr int kRowThreads = 256;
// Outputs that the L2s (8 x 4 MB) do not hold are written past them, which leaves those to what is read: a Q8_0 cache's
// 32048 tokens of 4 heads of 128 read back 24.8 -> 19.4 us.
constexpr uint64_t kStreamFrom = 32u << 20;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

// m cos and m sin of `turns` revolutions, each rounded once: the angle is cut to a quarter turn and the Taylor polynomials are summed in 64 bits (a position of 2^20 has
// 2^-4 radians left in 32; one thread does this for each pair of a token, all heads use it).  On [-pi/4, pi/4] the sine's next term is below 2^-37, the cosine's 2^-33.
__device__ __forceinline__ float2 cos_sin_turns(double turns, double m) {
    const double quarters = turns * 4.0, k = rint(quarters), a = (quarters - k) * 1.5707963267948966, a2 = a * a;
    double s = fma(a2, -1.0 / 39916800.0, 1.0 / 362880.0);
    s = fma(a2, s, -1.0 / 5040.0);
    s = fma(a2, s, 1.0 / 120.0);
    s = fma(a2, s, -1.0 / 6.0);
    s = fma(a * a2, s, a) * m;
    double c = fma(a2, -1.0 / 3628800.0, 1.0 / 40320.0);
    c = fma(a2, c, -1.0 / 720.0);
    c = fma(a2, c, 1.0 / 24.0);
    c = fma(a2, c, -0.5);
    c = fma(a2, c, 1.0) * m;
    const int q = (int)(k - 4.0 * floor(k * 0.25));
    const float cc = (float)((q & 1) ? s : c), ss = (float)((q & 1) ? c : s);
    return make_float2((q == 1 || q == 2) ? -cc : cc, (q & 2) ? -ss : ss);
}

struct RowsArgs {
    const half_t *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride, q_out_stride;
    half_t* q_out;
    void *k_cache, *v_cache;       // fp16, or int8
    half_t *k_d, *v_d;             // Q8_0 scales
    const int32_t *positions, *slots;
    const double* freqs;
    uint32_t Hq, Hkv, chunks, n_rot, heads_per_wg, groups, page_size, n_slots;  // chunks = D / 8, groups: workgroups of a token
    double mscale;
};

__device__ __forceinline__ uint32_t max_bits4(uint32_t v) {  // over four adjacent lanes
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}

// Eight elements of an interleaved chunk / the first and the second eight of a pair of chunks, turned by cs[0 ..]; products and sums in fp32, one rounding.
__device__ __forceinline__ half8 turn_interleaved(half8 x, const float2* cs) {
    half8 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 w = cs[i];
        const float x0 = (float)x[2 * i], x1 = (float)x[2 * i + 1];
        y[2 * i] = f32_to_f16_rne(fmaf(x0, w.x, -(x1 * w.y)));
        y[2 * i + 1] = f32_to_f16_rne(fmaf(x0, w.y, x1 * w.x));
    }
    return y;
}
__device__ __forceinline__ half8 turn_first(half8 x0, half8 x1, const float2* cs) {
    half8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = f32_to_f16_rne(fmaf((float)x0[i], cs[i].x, -((float)x1[i] * cs[i].y)));
    return y;
}
__device__ __forceinline__ half8 turn_second(half8 x0, half8 x1, const float2* cs) {
    half8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = f32_to_f16_rne(fmaf((float)x0[i], cs[i].y, (float)x1[i] * cs[i].x));
    return y;
}
__device__ __forceinline__ float2 cs_of(const RowsArgs& a, uint32_t t, uint32_t i) {
    return cos_sin_turns((double)a.positions[t] * (a.freqs[i] * 0.15915494309189535), a.mscale);
}
__device__ __forceinline__ const half_t* row_of(const RowsArgs& a, uint32_t t, uint32_t h, uint32_t D) {
    return h < a.Hq ? a.q + t * a.q_stride + (size_t)h * D : h < a.Hq + a.Hkv ? a.k + t * a.k_stride + (size_t)(h - a.Hq) * D : a.v + t * a.v_stride + (size_t)(h - a.Hq - a.Hkv) * D;
}

// Chunk c of head h (query, key, value heads in this order) of token t to where it goes.  Q8: the four lanes of a block of 32 call together.
template <bool Q8>
__device__ __forceinline__ void put(const RowsArgs& a, uint32_t t, uint32_t slot, uint32_t h, uint32_t c, half8 y) {
    const uint32_t D = a.chunks * 8;
    if (h < a.Hq) {
        *reinterpret_cast<half8*>(a.q_out + t * a.q_out_stride + (size_t)h * D + c * 8) = y;
        return;
    }
    if (slot >= a.n_slots) return;
    const bool is_v = h >= a.Hq + a.Hkv;
    const uint32_t hk = h - a.Hq - (is_v ? a.Hkv : 0), page = slot / a.page_size, at = slot - page * a.page_size;
    const size_t crow = ((size_t)page * a.Hkv + hk) * a.page_size + at;
    void* cache = is_v ? a.v_cache : a.k_cache;
    if (!Q8) {
        *reinterpret_cast<half8*>(static_cast<half_t*>(cache) + crow * D + c * 8) = y;
    } else {
        // the largest magnitude by its bits: a NaN's are above all others, so that it reaches the scale
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, f2u(fabsf((float)y[i])));
        const float amax = u2f(max_bits4(top)), inv = amax > 0.f ? 127.0f / amax : 0.f;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t)(round_away_i((float)y[i] * inv) & 0xFF) << (8 * (i % 4));
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(cache) + crow * D + c * 8) = make_uint2(w[0], w[1]);
        if ((c & 3) == 0) (is_v ? a.v_d : a.k_d)[crow * (D / 32) + c / 4] = f32_to_f16_rne(amax / 127.0f);
    }
}

// One workgroup takes heads_per_wg heads of one token, one thread 8 consecutive elements of a head.  A thread loads its own 8 and, in the half layout, the 8 that they
// are paired with before the barrier behind which the sines are ready, and stores after it: rows may be rotated in place.
template <bool ROPE, bool Q8, bool INTER>
__global__ __launch_bounds__(kRowThreads) void rows_kernel(RowsArgs a) {
    __shared__ float2 cs[128];
    const uint32_t tid = threadIdx.x, t = blockIdx.x / a.groups, D = a.chunks * 8;
    const uint32_t hw = tid / a.chunks, c = tid - hw * a.chunks, h = (blockIdx.x - t * a.groups) * a.heads_per_wg + hw;
    const bool live = hw < a.heads_per_wg && h < a.Hq + 2 * a.Hkv;
    half8 own = {}, other = {};
    const bool turned = ROPE && h < a.Hq + a.Hkv && c * 8 < a.n_rot;
    const uint32_t half_chunks = a.n_rot / 16;
    const bool first = c < half_chunks;
    if (live) {
        const half_t* row = row_of(a, t, h, D);
        own = *reinterpret_cast<const half8*>(row + c * 8);
        if (!INTER && turned) other = *reinterpret_cast<const half8*>(row + (first ? c + half_chunks : c - half_chunks) * 8);
    }
    const uint32_t slot = a.slots ? (uint32_t)a.slots[t] : 0u;
    if (ROPE) {
        if (tid < a.n_rot / 2) cs[tid] = cs_of(a, t, tid);
        __syncthreads();
    }
    if (!live) return;   // whole groups of four lanes: chunks % 4 == 0 wherever they exchange values
    half8 y = own;
    if (turned) y = INTER ? turn_interleaved(own, cs + c * 4) : first ? turn_first(own, other, cs + c * 8) : turn_second(other, own, cs + (c - half_chunks) * 8);
    put<Q8>(a, t, slot, h, c, y);
}

// Prompts: a workgroup takes one token with all its heads, a thread two chunks at a time, in the half layout the two that are turned together: rows may be rotated
// in place.  The chunks of a head that are not turned, and a value head's, are paired with the same distance between the two throughout.
// Q8: that distance is a multiple of four chunks (D and n_rot multiples of 64), so that four lanes hold whole blocks.
template <bool ROPE, bool Q8, bool INTER>
__global__ __launch_bounds__(kRowThreads) void prompt_kernel(RowsArgs a) {
    __shared__ float2 cs[128];
    const uint32_t tid = threadIdx.x, threads = blockDim.x, t = blockIdx.x, D = a.chunks * 8, pairs = a.chunks / 2, items = (a.Hq + 2 * a.Hkv) * pairs, half_chunks = a.n_rot / 16;
    struct Item {
        uint32_t h, c0, c1;
        bool together, angle;
        half8 x0, x1;
    };
    auto load = [&](uint32_t i) {
        Item m;
        m.h = i / pairs;
        const uint32_t p = i - m.h * pairs;
        m.angle = ROPE && m.h < a.Hq + a.Hkv;
        // (p, p + half_chunks) among the turned chunks of the half layout, then (p', p' + rest / 2) behind them
        m.together = !INTER && m.angle && p < half_chunks;
        m.c0 = !INTER && m.angle && !m.together ? p + half_chunks : p;
        m.c1 = m.c0 + (INTER || !m.angle ? pairs : m.together ? half_chunks : pairs - half_chunks);
        const half_t* row = row_of(a, t, m.h, D);
        m.x0 = *reinterpret_cast<const half8*>(row + m.c0 * 8);
        m.x1 = *reinterpret_cast<const half8*>(row + m.c1 * 8);
        return m;
    };
    Item next;
    if (tid < items) next = load(tid);
    const uint32_t slot = a.slots ? (uint32_t)a.slots[t] : 0u;
    if (ROPE) {
        for (uint32_t i = tid; i < a.n_rot / 2; i += threads) cs[i] = cs_of(a, t, i);
        __syncthreads();
    }
    for (uint32_t i = tid; i < items; i += threads) {
        const Item m = next;
        if (i + threads < items) next = load(i + threads);
        half8 y0 = m.x0, y1 = m.x1;
        if (m.together) {
            y0 = turn_first(m.x0, m.x1, cs + m.c0 * 8);
            y1 = turn_second(m.x0, m.x1, cs + m.c0 * 8);
        } else if (INTER && m.angle) {
            if (m.c0 * 8 < a.n_rot) y0 = turn_interleaved(m.x0, cs + m.c0 * 4);
            if (m.c1 * 8 < a.n_rot) y1 = turn_interleaved(m.x1, cs + m.c1 * 4);
        }
        put<Q8>(a, t, slot, m.h, m.c0, y0);
        put<Q8>(a, t, slot, m.h, m.c1, y1);
    }
}

// A launch holds fewer than 2^32 threads in a row of its grid.
static bool fits(uint64_t workgroups, uint32_t threads) { return workgroups * threads < (1ull << 32); }

constexpr uint32_t kPromptTokens = 512;
template <bool ROPE, bool Q8>
static int launch_rows(mx_stream_t s, RowsArgs a, uint32_t T, int interleaved) {
    a.heads_per_wg = kRowThreads / a.chunks;
    a.groups = (a.Hq + 2 * a.Hkv + a.heads_per_wg - 1) / a.heads_per_wg;
    // Two chunks a thread load every row once where the half layout's other form loads turned rows twice: 8192 tokens of 72 heads of 64 35.9 -> 26.6 us (5.7 TB/s),
    // 2047 tokens of 32 + 4 + 4 heads of 128 into a Q8_0 cache 14.5 -> 9.4; interleaved pairs are as fast either way.  Fewer tokens leave CUs without work: one
    // token 2.2 -> 2.8 us, 333 (18 heads of 256) 3.9 -> 4.1.
    if (T >= kPromptTokens && (!Q8 || (a.chunks % 8 == 0 && a.n_rot % 64 == 0))) {
        // as many waves as the token's pairs of chunks fill evenly
        const uint32_t items = (a.Hq + 2 * a.Hkv) * (a.chunks / 2), turns = (items + kRowThreads - 1) / kRowThreads, threads = ((items + turns - 1) / turns + 63) / 64 * 64;
        MX_REQUIRE_SHAPE(fits(T, threads));
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(T), dim3(threads), 0, as_stream(s), a);
            return launch_status();
        };
        return ROPE && interleaved ? launch(prompt_kernel<ROPE, Q8, ROPE>) : launch(prompt_kernel<ROPE, Q8, false>);
    }
    MX_REQUIRE_SHAPE(fits((uint64_t)a.groups * T, kRowThreads));
    const dim3 grid(a.groups * T);
    if (ROPE && interleaved) hipLaunchKernelGGL((rows_kernel<ROPE, Q8, ROPE>), grid, dim3(kRowThreads), 0, as_stream(s), a);
    else hipLaunchKernelGGL((rows_kernel<ROPE, Q8, false>), grid, dim3(kRowThreads), 0, as_stream(s), a);
    return launch_status();
}

// Reading back: a workgroup takes 16 tokens of one sequence (they lie in one page) and 1024 pieces of 8 elements of their keys and values, a thread four, which it
// requests before it writes the first (4 ragged sequences of 300 tokens with 8 heads of 128, with their write: 11.8 us one after the other, 6.3; long ones run at a
// copy's rate: 10 k tokens of them in 15.9 us, 5.1 TB/s).
// Tile numbers are dealt by floor(rows[b] / 16) + b, which leaves room for every sequence's ceil(length / 16).
constexpr int kReadPieces = 4;
template <bool Q8, bool STREAM>
__global__ __launch_bounds__(256) void kv_read_kernel(const void* k_cache, const half_t* k_d, const void* v_cache, const half_t* v_d, const int32_t* page_table,
                                                      uint32_t max_pages, const int32_t* rows, half_t* k_out, half_t* v_out, uint32_t total, uint32_t B,
                                                      uint32_t Hkv, uint32_t chunks, uint32_t n_pages, uint32_t page_size) {
    const uint32_t lane = threadIdx.x & 63u, tile = blockIdx.x;
    uint32_t lo = 0, n = B;
    while (n > 1) {   // the last b whose first tile is not behind this one: 64 candidates at a time
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const bool behind = i < n && (uint32_t)rows[lo + i] / 16 + lo + i <= tile;
        const uint32_t cnt = max(1u, (uint32_t)__popcll(__ballot(behind)));
        lo += (cnt - 1) * step;
        n = min(step, n - (cnt - 1) * step);
    }
    const uint32_t b = lo, row0 = (uint32_t)rows[b], end = min((uint32_t)rows[b + 1], total), first = row0 / 16 + b;
    if (tile < first || row0 >= end) return;
    const uint32_t t0 = (tile - first) * 16;
    if (t0 >= end - row0) return;
    const uint32_t count = min(16u, end - row0 - t0), col = t0 / page_size, D = chunks * 8;
    const uint32_t page = col < max_pages ? (uint32_t)page_table[(size_t)b * max_pages + col] : 0xFFFFFFFFu;
    const bool good = page < n_pages;
    const uint32_t per_head = 16 * chunks, items = 2 * Hkv * per_head, i0 = blockIdx.y * (256 * kReadPieces) + threadIdx.x;
    constexpr int U = kReadPieces;
    uint4 got[U];
    half_t d[U];
    uint32_t at[U];                      // token * heads * chunks + head * chunks + chunk, from the tile's first row
    bool is_v[U], live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t i = i0 + 256 * u, hh = i / per_head, r = i - hh * per_head, tok = r / chunks, c = r - tok * chunks;
        live[u] = i < items && tok < count;
        is_v[u] = hh >= Hkv;
        const uint32_t h = is_v[u] ? hh - Hkv : hh;
        at[u] = (tok * Hkv + h) * chunks + c;
        got[u] = make_uint4(0, 0, 0, 0);
        d[u] = (half_t)0.f;
        if (live[u] && good) {
            const size_t crow = ((size_t)page * Hkv + h) * page_size + (t0 - col * page_size) + tok;
            const void* cache = is_v[u] ? v_cache : k_cache;
            if (!Q8) {
                got[u] = *reinterpret_cast<const uint4*>(static_cast<const half_t*>(cache) + crow * D + c * 8);
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(cache) + crow * D + c * 8);
                got[u].x = w.x;
                got[u].y = w.y;
                d[u] = (is_v[u] ? v_d : k_d)[crow * (D / 32) + c / 4];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!live[u]) continue;
        half8 y = __builtin_bit_cast(half8, got[u]);
        if (Q8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = f32_to_f16_rne((float)(int8_t)((j < 4 ? got[u].x : got[u].y) >> (8 * (j & 3))) * (float)d[u]);
        }
        half8* const out = reinterpret_cast<half8*>((is_v[u] ? v_out : k_out) + (size_t)(row0 + t0) * Hkv * D) + at[u];
        if (STREAM) __builtin_nontemporal_store(y, out);
        else *out = y;
    }
}

// ---------------------------------------------------------------- argument checks (before any HIP call)
static int check_cache(bool q8, const void* k, const void* k_d, const void* v, const void* v_d, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size) {
    MX_REQUIRE_PTR(k); MX_REQUIRE_PTR(v);
    if (q8) { MX_REQUIRE_PTR(k_d); MX_REQUIRE_PTR(v_d); }
    MX_REQUIRE_SHAPE(Hkv > 0 && Hkv <= 65535 && D > 0 && D <= 256 && D % (q8 ? 32 : 16) == 0);
    MX_REQUIRE_SHAPE(n_pages > 0 && page_size > 0 && page_size % 16 == 0 && (uint64_t)n_pages * page_size < (1ull << 31));
    MX_REQUIRE_ALIGN(k, 16); MX_REQUIRE_ALIGN(v, 16);
    if (q8) { MX_REQUIRE_ALIGN(k_d, 16); MX_REQUIRE_ALIGN(v_d, 16); }
    return MX_OK;
}
static int check_rows(const void* p, uint64_t stride, uint64_t width) {
    MX_REQUIRE_PTR(p);
    MX_REQUIRE_SHAPE(stride % 8 == 0 && stride >= width);
    MX_REQUIRE_ALIGN(p, 16);
    return MX_OK;
}
// In place is row by row: the same rows with other strides lie in each other's way.
static int check_in_place(const void* from, uint64_t from_stride, const void* to, uint64_t to_stride, uint32_t T) {
    MX_REQUIRE_SHAPE(from != to || from_stride == to_stride || T == 1);
    return MX_OK;
}
static int check_rotation(const void* positions, const void* freqs, uint32_t D, uint32_t n_rot) {
    MX_REQUIRE_PTR(positions); MX_REQUIRE_PTR(freqs);
    MX_REQUIRE_SHAPE(n_rot >= 16 && n_rot <= D && n_rot % 16 == 0);
    MX_REQUIRE_ALIGN(positions, 4); MX_REQUIRE_ALIGN(freqs, 8);
    return MX_OK;
}

static int rope_kv_write(mx_stream_t s, bool q8, const uint16_t* q, uint64_t q_stride, const uint16_t* k, uint64_t k_stride, const uint16_t* v, uint64_t v_stride,
                         uint16_t* q_out, uint64_t q_out_stride, void* k_cache, uint16_t* k_d, void* v_cache, uint16_t* v_d, const int32_t* positions,
                         const int32_t* slots, const double* freqs, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_rot, int interleaved,
                         double mscale, uint32_t n_pages, uint32_t page_size) {
    if (int rc = check_cache(q8, k_cache, k_d, v_cache, v_d, Hkv, D, n_pages, page_size)) return rc;
    if (int rc = check_rows(k, k_stride, (uint64_t)Hkv * D)) return rc;
    if (int rc = check_rows(v, v_stride, (uint64_t)Hkv * D)) return rc;
    MX_REQUIRE_PTR(slots);
    MX_REQUIRE_ALIGN(slots, 4);
    MX_REQUIRE_SHAPE(T > 0 && Hq <= 65535);
    if (freqs) {
        MX_REQUIRE_SHAPE(Hq > 0);
        if (int rc = check_rows(q, q_stride, (uint64_t)Hq * D)) return rc;
        if (int rc = check_rows(q_out, q_out_stride, (uint64_t)Hq * D)) return rc;
        if (int rc = check_in_place(q, q_stride, q_out, q_out_stride, T)) return rc;
        if (int rc = check_rotation(positions, freqs, D, n_rot)) return rc;
    }
    RowsArgs a = {};
    a.q = reinterpret_cast<const half_t*>(q); a.k = reinterpret_cast<const half_t*>(k); a.v = reinterpret_cast<const half_t*>(v);
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.q_out_stride = q_out_stride;
    a.q_out = reinterpret_cast<half_t*>(q_out);
    a.k_cache = k_cache; a.v_cache = v_cache;
    a.k_d = reinterpret_cast<half_t*>(k_d); a.v_d = reinterpret_cast<half_t*>(v_d);
    a.positions = positions; a.slots = slots; a.freqs = freqs;
    a.Hq = Hq; a.Hkv = Hkv; a.chunks = D / 8; a.n_rot = n_rot; a.page_size = page_size; a.n_slots = n_pages * page_size;
    a.mscale = mscale;
    if (freqs) return q8 ? launch_rows<true, true>(s, a, T, interleaved) : launch_rows<true, false>(s, a, T, interleaved);
    return q8 ? launch_rows<false, true>(s, a, T, 0) : launch_rows<false, false>(s, a, T, 0);
}

static int kv_read(mx_stream_t s, bool q8, const void* k, const uint16_t* k_d, const void* v, const uint16_t* v_d, const int32_t* page_table, uint32_t max_pages,
                   const int32_t* rows, uint16_t* k_out, uint16_t* v_out, uint32_t total_rows, uint32_t B, uint32_t Hkv, uint32_t D, uint32_t n_pages,
                   uint32_t page_size) {
    if (int rc = check_cache(q8, k, k_d, v, v_d, Hkv, D, n_pages, page_size)) return rc;
    MX_REQUIRE_PTR(page_table); MX_REQUIRE_PTR(rows); MX_REQUIRE_PTR(k_out); MX_REQUIRE_PTR(v_out);
    MX_REQUIRE_SHAPE(B > 0 && B <= (1u << 24) && max_pages > 0 && total_rows > 0 && total_rows < (1u << 31) && fits(total_rows / 16 + (uint64_t)B, 256));
    MX_REQUIRE_ALIGN(page_table, 4); MX_REQUIRE_ALIGN(rows, 4); MX_REQUIRE_ALIGN(k_out, 16); MX_REQUIRE_ALIGN(v_out, 16);
    const dim3 grid(total_rows / 16 + B, (2 * Hkv * 16 * (D / 8) + 256 * kReadPieces - 1) / (256 * kReadPieces));
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(s), k, reinterpret_cast<const half_t*>(k_d), v, reinterpret_cast<const half_t*>(v_d), page_table,
                           max_pages, rows, reinterpret_cast<half_t*>(k_out), reinterpret_cast<half_t*>(v_out), total_rows, B, Hkv, D / 8, n_pages, page_size);
        return launch_status();
    };
    if ((uint64_t)total_rows * Hkv * D * 4 >= kStreamFrom) return q8 ? launch(kv_read_kernel<true, true>) : launch(kv_read_kernel<false, true>);
    return q8 ? launch(kv_read_kernel<true, false>) : launch(kv_read_kernel<false, false>);
}

}  // namespace mxq

using namespace mxq;

extern "C" {

int mx_rope_freqs(uint32_t n_rot, double base, double scale, double ext_factor, double attn_factor, double beta_fast, double beta_slow, uint32_t n_ctx_orig,
                  const float* factors, double* freqs, double* mscale) {
    MX_REQUIRE_PTR(freqs); MX_REQUIRE_PTR(mscale);
    const bool yarn = ext_factor != 0.0;
    MX_REQUIRE_SHAPE(n_rot >= 16 && n_rot <= 256 && n_rot % 16 == 0 && base > 1.0 && scale > 0.0 && ext_factor >= 0.0 && ext_factor <= 1.0);
    MX_REQUIRE_SHAPE(!yarn || (n_ctx_orig > 0 && beta_fast > 0.0 && beta_slow > 0.0 && beta_fast >= beta_slow));
    const double pi = 3.14159265358979323846, n = n_rot;
    auto dim = [&](double turns) { return n * log(n_ctx_orig / (turns * 2.0 * pi)) / (2.0 * log(base)); };
    const double low = yarn ? fmax(0.0, floor(dim(beta_fast))) : 0.0, high = yarn ? fmin(n - 1.0, ceil(dim(beta_slow))) : 0.0;
    for (uint32_t i = 0; i < n_rot / 2; ++i) {
        const double f = pow(base, -2.0 * i / n) / (factors ? (double)factors[i] : 1.0);
        const double keep = yarn ? ext_factor * (1.0 - fmin(1.0, fmax(0.0, (i - low) / fmax(0.001, high - low)))) : 0.0;
        freqs[i] = f * scale * (1.0 - keep) + f * keep;
    }
    *mscale = attn_factor * (yarn ? 1.0 + 0.1 * log(1.0 / scale) : 1.0);
    return MX_OK;
}

int mx_rope(mx_stream_t s, const uint16_t* x, uint64_t x_stride, uint16_t* y, uint64_t y_stride, const int32_t* positions, const double* freqs, uint32_t T,
            uint32_t n_heads, uint32_t D, uint32_t n_rot, int interleaved, double mscale) {
    MX_REQUIRE_SHAPE(T > 0 && n_heads > 0 && n_heads <= 65535 && D > 0 && D <= 256 && D % 16 == 0);
    if (int rc = check_rows(x, x_stride, (uint64_t)n_heads * D)) return rc;
    if (int rc = check_rows(y, y_stride, (uint64_t)n_heads * D)) return rc;
    if (int rc = check_in_place(x, x_stride, y, y_stride, T)) return rc;
    if (int rc = check_rotation(positions, freqs, D, n_rot)) return rc;
    RowsArgs a = {};
    a.q = reinterpret_cast<const half_t*>(x); a.q_out = reinterpret_cast<half_t*>(y);
    a.q_stride = x_stride; a.q_out_stride = y_stride;
    a.positions = positions; a.freqs = freqs;
    a.Hq = n_heads; a.chunks = D / 8; a.n_rot = n_rot; a.mscale = mscale;
    return launch_rows<true, false>(s, a, T, interleaved);
}

int mx_rope_kv_write_f16(mx_stream_t s, const uint16_t* q, uint64_t q_stride, const uint16_t* k, uint64_t k_stride, const uint16_t* v, uint64_t v_stride,
                         uint16_t* q_out, uint64_t q_out_stride, uint16_t* k_cache, uint16_t* v_cache, const int32_t* positions, const int32_t* slots,
                         const double* freqs, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_rot, int interleaved, double mscale,
                         uint32_t n_pages, uint32_t page_size) {
    MX_REQUIRE_PTR(freqs);
    return rope_kv_write(s, false, q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, k_cache, nullptr, v_cache, nullptr, positions, slots, freqs, T, Hq,
                         Hkv, D, n_rot, interleaved, mscale, n_pages, page_size);
}
int mx_rope_kv_write_q8_0(mx_stream_t s, const uint16_t* q, uint64_t q_stride, const uint16_t* k, uint64_t k_stride, const uint16_t* v, uint64_t v_stride,
                          uint16_t* q_out, uint64_t q_out_stride, int8_t* k_qs, uint16_t* k_d, int8_t* v_qs, uint16_t* v_d, const int32_t* positions,
                          const int32_t* slots, const double* freqs, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_rot, int interleaved,
                          double mscale, uint32_t n_pages, uint32_t page_size) {
    MX_REQUIRE_PTR(freqs);
    return rope_kv_write(s, true, q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, k_qs, k_d, v_qs, v_d, positions, slots, freqs, T, Hq, Hkv, D, n_rot,
                         interleaved, mscale, n_pages, page_size);
}
int mx_kv_write_f16(mx_stream_t s, const uint16_t* k, uint64_t k_stride, const uint16_t* v, uint64_t v_stride, uint16_t* k_cache, uint16_t* v_cache,
                    const int32_t* slots, uint32_t T, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size) {
    return rope_kv_write(s, false, nullptr, 0, k, k_stride, v, v_stride, nullptr, 0, k_cache, nullptr, v_cache, nullptr, nullptr, slots, nullptr, T, 0, Hkv, D, 0, 0,
                         1.0, n_pages, page_size);
}
int mx_kv_write_q8_0(mx_stream_t s, const uint16_t* k, uint64_t k_stride, const uint16_t* v, uint64_t v_stride, int8_t* k_qs, uint16_t* k_d, int8_t* v_qs,
                     uint16_t* v_d, const int32_t* slots, uint32_t T, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size) {
    return rope_kv_write(s, true, nullptr, 0, k, k_stride, v, v_stride, nullptr, 0, k_qs, k_d, v_qs, v_d, nullptr, slots, nullptr, T, 0, Hkv, D, 0, 0, 1.0, n_pages,
                         page_size);
}
int mx_kv_read_f16(mx_stream_t s, const uint16_t* k_cache, const uint16_t* v_cache, const int32_t* page_table, uint32_t max_pages, const int32_t* rows,
                   uint16_t* k_out, uint16_t* v_out, uint32_t total_rows, uint32_t B, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size) {
    return kv_read(s, false, k_cache, nullptr, v_cache, nullptr, page_table, max_pages, rows, k_out, v_out, total_rows, B, Hkv, D, n_pages, page_size);
}
int mx_kv_read_q8_0(mx_stream_t s, const int8_t* k_qs, const uint16_t* k_d, const int8_t* v_qs, const uint16_t* v_d, const int32_t* page_table,
                    uint32_t max_pages, const int32_t* rows, uint16_t* k_out, uint16_t* v_out, uint32_t total_rows, uint32_t B, uint32_t Hkv, uint32_t D,
                    uint32_t n_pages, uint32_t page_size) {
    return kv_read(s, true, k_qs, k_d, v_qs, v_d, page_table, max_pages, rows, k_out, v_out, total_rows, B, Hkv, D, n_pages, page_size);
}

}  // extern "C"
