// attn_decode.hip — attention of one new token over a paged key-value cache (fp16 or Q8_0 planes).
#include "mxq_device.h"
#include "mxq_host.h"

namespace mxq {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kTile = 32, kWaves = 4, kLeastShare = kWaves;   // tokens of a tile, waves of a workgroup, tiles of a share at least
constexpr float kShift = 15.f, kMostShifted = 1 << 20;   // what a running maximum lies below the largest score, scores for which it does (log2 units)
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
    const half_t* q;
    uint64_t q_stride;
    const void *k, *v;              // fp16, or int8
    const half_t *k_d, *v_d;        // Q8_0 scales
    const int32_t *table, *lens;
    const float* sinks;
    half_t* out;
    uint8_t* out_q8;
    float *part_o, *part_ml;        // parts of sequences: [part][Hq][D] sums and [part][Hq] (maximum, sum of weights)
    uint32_t* parts;                // [B] (first part, how many)
    uint32_t B, Hq, Hkv, D, max_pages, n_pages, page_size, page_shift, window, shares;   // page_shift: log2 of a page size that is a power of two, else 32
    float scale;                    // times log2(e)
};

// The tokens of a sequence: [start, end), in tiles of 32 that begin at multiples of 32.
struct Span {
    uint32_t start, end, tile0, tiles;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int32_t len) {
    const uint64_t capacity = (uint64_t)a.max_pages * a.page_size;
    Span s;
    s.end = len <= 0 ? 0u : (uint32_t)min((uint64_t)len, capacity);
    s.start = a.window && s.end > a.window ? s.end - a.window : 0u;
    s.tile0 = s.start / kTile;
    s.tiles = s.end ? (s.end - 1) / kTile + 1 - s.tile0 : 0u;
    return s;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);    // row_shr:1, 2, 4, 8 within 16 lanes
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);   // the last lane of rows 0 and 2 to rows 1 and 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);   // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }

// Equal shares: the tiles of all sequences in a row, cut into `shares` ranges of `per` tiles (at least kLeastShare).  A workgroup's range may end one sequence
// and begin another; its part of sequence b has the number share + b, which no other part has, and the parts of one sequence are consecutive.
struct Share {
    uint32_t per, left;      // tiles of a share; of this one
    uint32_t b, from;        // the sequence that it begins in, and at which of its tiles
    int32_t len;             // that sequence's entry
};
__device__ __forceinline__ Share share_of(const AttnArgs& a, uint32_t share, uint32_t lane) {
    uint32_t total = 0, upto = 0, own = 0;
    int32_t len = 0;
    for (uint32_t i0 = 0; i0 < a.B; i0 += 64) {
        len = i0 + lane < a.B ? a.lens[i0 + lane] : 0;
        own = span_of(a, len).tiles;
        if (own == 0 && i0 + lane < a.B && share == 0 && blockIdx.y == 0)
            *reinterpret_cast<uint2*>(a.parts + 2 * (i0 + lane)) = make_uint2(0, 0);   // no part: zeros, whatever the sinks
        upto = lanes_upto(own);
        total += lane_value(upto, 63);
    }
    Share s;
    s.per = max(kLeastShare, (total + a.shares - 1) / a.shares);
    const uint64_t at = (uint64_t)share * s.per;
    s.left = at < total ? min(s.per, total - (uint32_t)at) : 0u;
    s.b = s.from = 0;
    s.len = 0;
    uint32_t before = 0;
    for (uint32_t i0 = 0; s.left && i0 < a.B; i0 += 64) {
        if (a.B > 64) {      // up to 64 sequences: as they were
            len = i0 + lane < a.B ? a.lens[i0 + lane] : 0;
            own = span_of(a, len).tiles;
            upto = lanes_upto(own);
        }
        const uint64_t hit = __ballot(before + upto > (uint32_t)at);
        if (hit) {
            const int first = __ffsll((unsigned long long)hit) - 1;
            s.b = i0 + first;
            s.from = (uint32_t)at - before - lane_value(upto - own, first);
            s.len = (int32_t)lane_value((uint32_t)len, first);
            break;
        }
        before += lane_value(upto, 63);
    }
    return s;
}

// Final rows: four consecutive elements of a thread's, all of 8 threads in one block of 32 (D % 32 == 0 where a stream is wanted).
__device__ __forceinline__ void store_rows(const AttnArgs& a, size_t at, const float (&o)[4], bool live) {
    half_t h[4];
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = f32_to_f16_rne(o[i]);
        v[i] = (float)h[i];
    }
    if (live) *reinterpret_cast<uint2*>(a.out + at) = *reinterpret_cast<const uint2*>(h);
    if (a.out_q8) emit_q8_1x(v, threadIdx.x & 7u, live, a.out_q8 + at / 32 * kQ81xBytes);
}

// The cache is read once: its lines need not stay.
template <class T>
__device__ __forceinline__ T load_once(const void* p) {
    typedef uint32_t vec __attribute__((ext_vector_type(sizeof(T) / 4)));
    return __builtin_bit_cast(T, __builtin_nontemporal_load(reinterpret_cast<const vec*>(p)));
}

// Largest / sum over the four 16-lane rows of a wave, in every lane: permlane swaps bring the other rows' values.
__device__ __forceinline__ float rows_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    v = fmaxf(u2f(r[0]), u2f(r[1]));
    r = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return fmaxf(u2f(r[0]), u2f(r[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    v = u2f(r[0]) + u2f(r[1]);
    r = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return u2f(r[0]) + u2f(r[1]);
}

// What a wave's lanes wrote to LDS is there for its other lanes: one wave's LDS accesses keep their order, so only the compiler is told.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ uint32_t pick(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
// Two unsigned bytes u (bytes `sel` of w) as the fp16 pair u - 128: 0x6400 + u is 1024 + u.
__device__ __forceinline__ half2_t bytes_f16(uint32_t w, uint32_t sel) {
    const half2_t bias = {(half_t)-1152.f, (half_t)-1152.f};
    return __builtin_bit_cast(half2_t, pick(w, 0x64646464u, sel)) + bias;
}

// Four sums of which some are NaN, over fp16 values.  An infinity times a weight's part, or times what a running sum is scaled by, is NaN where that is zero or where the two
// parts differ in sign: what is NaN is made again of the values alone that are no numbers, each once, so that infinities of one sign give one and others NaN.  (A weight that is
// NaN is in the sum of weights too.)  v: the elements in token 0 of head 0 of page 0.  A function of its own, since its registers would cost every call 2 % of a short sequence.
__device__ __attribute__((noinline)) floatx4 without_numbers(floatx4 sum, const half_t* v, const int32_t* table, uint32_t n_pages, uint32_t page_size, uint32_t hk, uint32_t Hkv, uint32_t D,
                                                             uint32_t from, uint32_t to) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = sum[j] == sum[j] ? sum[j] : 0.f;
    for (uint32_t t0 = from / 8 * 8; t0 < to; t0 += 8) {      // 8 tokens, of one page
        const uint32_t col = t0 / page_size, page = (uint32_t)table[col];
        if (page >= n_pages) continue;
        const half_t* row = v + (((size_t)page * Hkv + hk) * page_size + t0 - col * page_size) * D;
        uint2 w[8];
#pragma unroll
        for (uint32_t t = 0; t < 8; ++t) w[t] = *reinterpret_cast<const uint2*>(row + t * D);
#pragma unroll
        for (uint32_t t = 0; t < 8; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t bits = (j < 2 ? w[t].x : w[t].y) >> (16 * (j & 1)) & 0xFFFFu;
                if (t0 + t >= from && t0 + t < to && (bits & 0x7C00u) == 0x7C00u) sum[j] += h2f(bits);
            }
    }
    return sum;
}

// Scales of at most 511.5, whose products with -128 .. 127 fp16 holds.  Their bits' order as signed integers is theirs as numbers; a NaN may become 511.5.
__device__ __forceinline__ half8 at_most_511(half8 d) {
    typedef short short8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(half8, __builtin_elementwise_min(__builtin_bit_cast(short8, d), (short8)(short)0x5FFE));
}

// A workgroup takes one key-value head, up to 16 of the query heads that share it, and a sequence or a share of the sequences' tiles; its waves take the tiles in turn,
// each with a running maximum and sum of its own.  Bound by the cache's bytes: 64 x 8192 fp16 tokens of 8 heads of 128 in 322 us one after another,
// 6.7 TB/s, 328 to 334 each by itself under the tracer (a plain copy of that size moves 4.95, reads alone reach 6.3 to 7.1); what a launch has beside them is 5 us from its start to its first tile and from its last one to its end.
//
// Scores: S^T[token][head] = K Q^T, mfma 16x16x32.  Keys come in whole rows, 16 bytes a lane (read as the operand wants them, 16 rows a load, they kept the address units
// busy: Q8_0 99 -> 56 us for one sequence of 131071), and reach the operand through an LDS tile of the wave's own.  Row r of the two 16-row products of a tile is
// token 8 (r / 4) + r % 4 (+ 4), so that a lane, which gets 4 rows of a product, ends up with the 8 consecutive tokens 8g .. 8g + 7 of one head (g = lane / 16): exactly
// the operand layout of the second product, O^T[d][head] += V^T P^T, whose other operand is 8 tokens of one d a lane.  A lane loads elements E c .. E c + E - 1 (c = lane % 16,
// E = DP / 16) of its 8 tokens, whole rows by 16 lanes, and turns them in registers by byte permutes.
//
// Only the result is rounded to fp16: scores, maxima and sums are fp32, and the matrix instruction's fp16 operands carry the weights in two parts, the second what the first's
// rounding left (to 2^-22, or 2^-40 of the largest weight: that is 2^15, not 1, so that the many small weights of a long sequence lie above fp16's smallest step; where
// scores are so large that 15 of them could round to 16, it is 1).  Q8_0: keys are exact as fp16 integers and their scales are folded into the fp32 products of each block; values are q d in two parts, which hold it
// exactly (8 + 11 bits; d and so q d are multiples of 2^-24; the first part is that of a scale of at most 511.5, since 127 * 516, as which 65504 is stored, passes fp16: 64960 and
// 572).  One part would be 3 % faster and 1.4 times as far off.
// Registers: narrow Q8_0 heads take at most 128, so that four workgroups fit a CU (with 130: 126 sequences of up to 60 tokens of 8 heads of 64 6.5 -> 8.7 us).
template <bool Q8, int DP, int NBLK, bool FULL>
__global__ __launch_bounds__(kWaves * 64, DP == 256 ? (Q8 ? 2 : 1) : Q8 && DP == 64 ? 4 : FULL || Q8 ? 3 : 2) void attn_decode_kernel(AttnArgs a) {
    constexpr int E = DP / 16, NB = DP / 32;
    constexpr int VW = Q8 ? E / 4 : E / 2;                     // dwords of a lane's part of one value row, in VP pieces (wide fp16 heads: 8 of each half)
    constexpr int VP = !Q8 && E == 16 ? 2 : 1;
    constexpr int CPR = DP / (Q8 ? 16 : 8), RPI = 64 / CPR, KI = kTile / RPI;   // 16-byte pieces of a key row, rows of a load, loads of a tile
    constexpr int OS = DP + 4;                                  // LDS row stride of the waves' sums
    constexpr uint32_t ROW = CPR * 16;
    constexpr uint32_t SCALES = Q8 ? kTile * NBLK * 2 : 0, WAVE = kTile * ROW + 2 * SCALES;   // LDS of a wave: keys, their scales [token][block], the values' [block][token]
    extern __shared__ float lds[];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15u, g = lane >> 4;
    const uint32_t G = a.Hq / a.Hkv, tiles_of_heads = (G + 15) / 16;
    const uint32_t hk = blockIdx.y / tiles_of_heads, head0 = (blockIdx.y - hk * tiles_of_heads) * 16, heads = min(16u, G - head0);
    const uint32_t D = FULL ? (Q8 ? NBLK * 32 : DP) : Q8 ? NBLK * 32 : a.D;
    const bool shared = a.shares != 0;
    const uint32_t share = blockIdx.x;
    Share sh = {1, 1, blockIdx.x, 0, 0};
    if (shared) sh = share_of(a, share, lane);
    else sh.len = a.lens[sh.b];
    uint32_t b = sh.b, first = sh.from, left = sh.left;
    int32_t len = __builtin_amdgcn_readfirstlane(sh.len);
    for (; left; len = __builtin_amdgcn_readfirstlane(left ? a.lens[b + 1] : 0), ++b) {
    const Span sp = span_of(a, len);
    const uint32_t last = shared ? min(sp.tiles, first + left) : sp.tiles;
    const bool whole = first == 0 && last == sp.tiles;     // the result itself, not a part of it
    const size_t out0 = ((size_t)b * a.Hq + hk * G + head0) * D;
    if (shared) {
        if (sp.tiles == 0) continue;
        if (first == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
            // the first tile is tile per - left of the share; the last share may be shorter, but what begins in it ends in it
            *reinterpret_cast<uint2*>(a.parts + 2 * b) = make_uint2(share + b, (sh.per - left + sp.tiles - 1) / sh.per + 1);
        }
        left -= last - first;
    } else {
        left = 0;
    }

    // queries: in registers, or (wide heads, whose other operands fill them) in LDS behind the waves' tiles, the same for every wave
    constexpr bool QL = DP > 128;
    half8 qf[QL ? 1 : NB];
    half8* const ql = reinterpret_cast<half8*>(reinterpret_cast<char*>(lds) + kWaves * WAVE) + lane;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        half8 q = {};
        const uint32_t d = n * 32 + g * 8;
        if (r < heads && d < D) q = *reinterpret_cast<const half8*>(a.q + b * a.q_stride + (size_t)(hk * G + head0 + r) * D + d);
        if (QL) ql[n * 64] = q;        // every wave writes the same values
        else qf[QL ? 0 : n] = q;
    }

    typedef const __attribute__((address_space(4))) int32_t* table_t;
    const table_t table = (table_t)(uintptr_t)(a.table + (size_t)b * a.max_pages);
    struct Ref {             // a tile's first token and, for its two halves, page and place in the page
        uint32_t token, page[2], off[2];
    };
    auto page_of = [&](uint32_t t) { return a.page_shift < 32 ? t >> a.page_shift : t / a.page_size; };
    auto locate = [&](uint32_t tile) {
        Ref f;
        f.token = (sp.tile0 + tile) * kTile;
        const uint32_t c0 = page_of(f.token), o0 = f.token - c0 * a.page_size;
        const bool next = o0 + 16 >= a.page_size;
        const uint32_t c1 = next ? c0 + 1 : c0;
        f.off[0] = o0;
        f.off[1] = next ? 0 : o0 + 16;
        f.page[0] = (uint32_t)table[c0];                          // c0 < max_pages: the tile's first token is in front of the sequence's end
        f.page[1] = (uint32_t)table[min(c1, a.max_pages - 1)];
        return f;
    };
    auto row_of = [&](const Ref& f, int h) { return ((size_t)(f.page[h] < a.n_pages ? f.page[h] : 0u) * a.Hkv + hk) * a.page_size + f.off[h]; };

    uint32_t kr[KI][4], vr[8][VW];
    constexpr int SL = (16 * NBLK + 63) / 64;                 // dwords of a tile's scales in a lane
    uint32_t ks[SL], vs[SL];
    // keys: whole rows by CPR lanes each, into the wave's LDS tile, where a row's pieces lie permuted (piece p at p ^ f, f = row % 4 + 4 (row / 8 % 2), which
    // is lane % 8 of its reader), so that the 16 lanes that read the same piece of 16 rows meet different banks
    char* const keys = reinterpret_cast<char*>(lds) + wave * WAVE;
    half_t* const k_scales = reinterpret_cast<half_t*>(keys + kTile * ROW);
    half_t* const v_scales = reinterpret_cast<half_t*>(keys + kTile * ROW + SCALES);
    const uint32_t lr = lane / CPR, lp = lane % CPR, v_in = 8 * (g & 1u) * D + r * (E / VP);
    auto load_k = [&](const Ref& f) {
        const size_t row0 = row_of(f, 0), row1 = row_of(f, 1);
        if (FULL || lp * 16 < D * (Q8 ? 1 : 2)) {
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                const char* base = static_cast<const char*>(a.k) + (i * RPI >= 16 ? row1 : row0) * D * (Q8 ? 1 : 2);
                *reinterpret_cast<uint4*>(kr[i]) = load_once<uint4>(base + ((i * RPI & 15) + lr) * D * (Q8 ? 1 : 2) + lp * 16);
            }
        }
    };
    auto load_scales = [&](const Ref& f) {
        const size_t row0 = row_of(f, 0), row1 = row_of(f, 1);
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const uint32_t w = i * 64 + lane;          // 8 * NBLK dwords of each half
            if (SL * 64 == 16 * NBLK || w < 16 * NBLK) {
                const size_t at = w < 8 * NBLK ? row0 * NBLK + 2 * w : row1 * NBLK + 2 * (w - 8 * NBLK);
                ks[i] = *reinterpret_cast<const uint32_t*>(a.k_d + at);
                vs[i] = *reinterpret_cast<const uint32_t*>(a.v_d + at);
            }
        }
    };
    auto stage_scales = [&]() {
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const uint32_t w = i * 64 + lane;
            if (SL * 64 == 16 * NBLK || w < 16 * NBLK) {
                reinterpret_cast<uint32_t*>(k_scales)[w] = ks[i];
                const uint32_t t0 = 2 * w / NBLK, n0 = 2 * w % NBLK, t1 = (2 * w + 1) / NBLK, n1 = (2 * w + 1) % NBLK;
                reinterpret_cast<uint16_t*>(v_scales)[n0 * kTile + t0] = (uint16_t)vs[i];
                reinterpret_cast<uint16_t*>(v_scales)[n1 * kTile + t1] = (uint16_t)(vs[i] >> 16);
            }
        }
    };
    auto stage_k = [&]() {
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            const uint32_t row = i * RPI + lr, f = ((row & 3u) | (row >> 1 & 4u)) & (CPR - 1);
            *reinterpret_cast<uint4*>(keys + row * ROW + (lp ^ f) * 16) = *reinterpret_cast<const uint4*>(kr[i]);
        }
    };
    const char* const key_row = keys + (8 * (r >> 2) + (r & 3u)) * ROW;
    auto load_v = [&](const Ref& f) {
        const size_t row0 = row_of(f, 0), row1 = row_of(f, 1), at = (g >> 1 ? row1 : row0) * D + v_in;
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int w = 0; w < VP; ++w) {
                if (!FULL && w * 128 + r * (E / VP) >= D) continue;
                const char* p = static_cast<const char*>(a.v) + (at + t * D + w * 128) * (Q8 ? 1 : 2);
                if (VW == 1) vr[t][0] = load_once<uint32_t>(p);
                else if (VW == 2) *reinterpret_cast<uint2*>(vr[t]) = load_once<uint2>(p);
                else *reinterpret_cast<uint4*>(vr[t] + 4 * w) = load_once<uint4>(p);
            }
    };
    if (!FULL) {   // lanes behind the head's end load nothing
#pragma unroll
        for (int i = 0; i < KI; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) kr[i][w] = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[t][w] = 0;
    }

    float m = -INFINITY, l = 0.f;
    floatx4 o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = floatx4{0.f, 0.f, 0.f, 0.f};

    uint32_t tile = first + wave;
    if (tile < last) {
        Ref cur = locate(tile), next = cur;
        load_k(cur);
        if (Q8) load_scales(cur);
        load_v(cur);
        if (tile + kWaves < last) next = locate(tile + kWaves);
#pragma unroll 1
        for (; tile < last; tile += kWaves) {
            const bool more = tile + kWaves < last;
            // ---- scores
            wave_sync();                     // the tile before has been read
            stage_k();
            if (Q8) stage_scales();
            wave_sync();
            if (more) {
                load_k(next);
                if (Q8) load_scales(next);
            }
            float x[8];
            floatx4 score[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            uint32_t kd[2][2 * NBLK];       // scales of the lane's 4 tokens of either product
#pragma unroll
            for (int t = 0; Q8 && t < 2; ++t)
#pragma unroll
                for (int n = 0; n < NBLK; ++n) *reinterpret_cast<uint2*>(kd[t] + 2 * n) = reinterpret_cast<const uint2*>(k_scales + (8 * g + 4 * t) * NBLK)[n];
#pragma unroll
            for (int n = 0; n < (Q8 ? NBLK : NB); ++n) {
                const uint32_t f = (r & 7u) & (CPR - 1);
                const half8 q = QL ? ql[n * 64] : qf[QL ? 0 : n];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (Q8) {
                        const uint2 kw = *reinterpret_cast<const uint2*>(key_row + t * 4 * ROW + ((2 * n + (g >> 1)) ^ f) * 16 + 8 * (g & 1u));
                        half8 kf;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const half2_t h = bytes_f16((w < 2 ? kw.x : kw.y) ^ 0x80808080u, w & 1 ? 0x00070006u : 0x00050004u);
                            kf[2 * w] = h[0];
                            kf[2 * w + 1] = h[1];
                        }
                        const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
                        const floatx4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q, zero, 0, 0, 0);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = j * NBLK + n;
                            score[t][j] = fmaf(p[j], h2f((i & 1 ? kd[t][i / 2] >> 16 : kd[t][i / 2]) & 0xFFFFu), score[t][j]);
                        }
                    } else {
                        score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const half8*>(key_row + t * 4 * ROW + ((4 * n + g) ^ f) * 16), q, score[t], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = score[i / 4][i % 4] * a.scale;
            const bool ok0 = cur.page[0] < a.n_pages, ok1 = cur.page[1] < a.n_pages, full = cur.token >= sp.start && cur.token + kTile <= sp.end && ok0 && ok1;
            half8 sc = {};       // scales of the lane's 8 values' block
            if (Q8) sc = *reinterpret_cast<const half8*>(v_scales + min(r * E / 32, NBLK - 1u) * kTile + 8 * g);
            if (!full) {   // masked tokens: no weight, and values of zero, since what lies there may be no number
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t t = cur.token + 8 * g + i;
                    const bool ok = t >= sp.start && t < sp.end && (g >> 1 ? ok1 : ok0);
                    x[i] = ok ? x[i] : -INFINITY;
                    sc[i] = ok ? sc[i] : (half_t)0.f;
#pragma unroll
                    for (int w = 0; w < VW; ++w) vr[i][w] = ok ? vr[i][w] : 0u;
                }
            }
            // ---- running maximum and sum
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            top = rows_max(top);
            top = fmaxf(m, fabsf(top) < kMostShifted ? top - kShift : top);
            const float ref = top == -INFINITY ? 0.f : top;
            if (__any(top > m)) {
                const float keep = __builtin_amdgcn_exp2f(m - ref);
                l *= keep;
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[e][j] *= keep;
                m = top;
            }
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = __builtin_amdgcn_exp2f(x[i] - ref);
                l += p;
                hi[i] = (half_t)p;
                lo[i] = (half_t)(p - (float)hi[i]);
            }
            // ---- values
            const half8 sm = at_most_511(sc);       // of the first parts
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                half8 f0, f1, g0, g1;   // elements e and e + 1 of 8 tokens; Q8_0: what their rounding to fp16 left
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    half2_t h0, h1;
                    if (Q8) {
                        const uint32_t both = pick(vr[2 * w + 1][e / 4] , vr[2 * w][e / 4], e & 2 ? 0x07030602u : 0x05010400u) ^ 0x80808080u;
                        const half2_t d = {sc[2 * w], sc[2 * w + 1]}, q0 = bytes_f16(both, 0x00050004u), q1 = bytes_f16(both, 0x00070006u);
                        h0 = q0 * half2_t{sm[2 * w], sm[2 * w + 1]};
                        h1 = q1 * half2_t{sm[2 * w], sm[2 * w + 1]};
                        const half2_t l0 = __builtin_elementwise_fma(q0, d, -h0), l1 = __builtin_elementwise_fma(q1, d, -h1);
                        g0[2 * w] = l0[0]; g0[2 * w + 1] = l0[1];
                        g1[2 * w] = l1[0]; g1[2 * w + 1] = l1[1];
                    } else {
                        h0 = __builtin_bit_cast(half2_t, pick(vr[2 * w + 1][e / 2], vr[2 * w][e / 2], 0x05040100u));
                        h1 = __builtin_bit_cast(half2_t, pick(vr[2 * w + 1][e / 2], vr[2 * w][e / 2], 0x07060302u));
                    }
                    f0[2 * w] = h0[0]; f0[2 * w + 1] = h0[1];
                    f1[2 * w] = h1[0]; f1[2 * w + 1] = h1[1];
                }
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f0, hi, o[e], 0, 0, 0);
                o[e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f1, hi, o[e + 1], 0, 0, 0);
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f0, lo, o[e], 0, 0, 0);
                o[e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f1, lo, o[e + 1], 0, 0, 0);
                if (Q8) {
                    o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(g0, hi, o[e], 0, 0, 0);
                    o[e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(g1, hi, o[e + 1], 0, 0, 0);
                }
            }
            if (more) {
                load_v(next);
                cur = next;
                if (tile + 2 * kWaves < last) next = locate(tile + 2 * kWaves);
            }
        }
    }

    // ---- the waves' sums: lane (r, g) holds elements 4 E g .. 4 E g + 4 E - 1 of head r
    l = rows_sum(l);
    __syncthreads();                         // the key tiles' place is taken
    float* ml = lds;                         // [waves][16] (maximum, sum)
    float* os = lds + kWaves * 32;            // [waves][heads][OS]
    if (g == 0) {
        ml[(wave * 16 + r) * 2] = m;
        ml[(wave * 16 + r) * 2 + 1] = l;
    }
    if (r < heads) {
        float* row = os + (wave * heads + r) * OS + 4 * (E / VP) * g;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<floatx4*>(row + (E / VP) * j + e / (E / VP) * 128 + e % (E / VP)) = floatx4{o[e][j], o[e + 1][j], o[e + 2][j], o[e + 3][j]};
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x * 4; i < (heads * D + kWaves * 256 - 1) / (kWaves * 256) * (kWaves * 256); i += kWaves * 256) {
        const bool live = i < heads * D;
        const uint32_t h = live ? i / D : 0, d = live ? i - h * D : 0;
        const uint32_t hq = hk * G + head0 + h;
        const float sink = whole && a.sinks ? a.sinks[hq] * kLog2e : -INFINITY;
        float top = sink, total = 0.f;
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * 16 + h) * 2]);
        const float ref = top == -INFINITY ? 0.f : top;
        floatx4 sum = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[(w * 16 + h) * 2] - ref);
            total += f * ml[(w * 16 + h) * 2 + 1];
            sum += f * *reinterpret_cast<const floatx4*>(os + (w * heads + h) * OS + d);
        }
        const float four = sum[0] + sum[1] + sum[2] + sum[3];
        if (!Q8 && __builtin_expect(four != four, 0)) {
            sum = without_numbers(sum, static_cast<const half_t*>(a.v) + d, a.table + (size_t)b * a.max_pages, a.n_pages, a.page_size, hk, a.Hkv, D, max(sp.start, (sp.tile0 + first) * kTile),
                                  min(sp.end, (sp.tile0 + last) * kTile));
            total = total == 0.f ? 0x1p-126f : total;   // however little weight a sink has left the tokens
        }
        if (whole) {
            const float all = total + __builtin_amdgcn_exp2f(sink - ref), inv = 1.0f / all;
            const bool none = total == 0.f;
            const float y[4] = {none ? 0.f : sum[0] * inv, none ? 0.f : sum[1] * inv, none ? 0.f : sum[2] * inv, none ? 0.f : sum[3] * inv};
            store_rows(a, out0 + i, y, live);
        } else if (live) {
            const size_t at = (size_t)(share + b) * a.Hq + hq;
            *reinterpret_cast<floatx4*>(a.part_o + at * D + d) = sum;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(top, total);
        }
    }
    first = 0;
    if (left) __syncthreads();               // the sums have been read
    }
}

// A part's weight in the sum of parts, never zero: an infinite sum stays one.  (What 2^-126 of a finite one adds is far below fp16.)
__device__ __forceinline__ float part_weight(float x) { return fmaxf(__builtin_amdgcn_exp2f(x), 0x1p-126f); }
// The result: zero where no token has a weight, an infinity all the same.
__device__ __forceinline__ float divided(float sum, float total, float inv) { return total == 0.f && fabsf(sum) < INFINITY ? 0.f : sum * inv; }

// Joins the parts of one head of one sequence: D / 4 threads for each of `groups` groups of parts, each thread four elements.
__global__ __launch_bounds__(512) void attn_join_kernel(AttnArgs a, uint32_t groups) {
    extern __shared__ float sums[];          // [groups][D]
    const uint32_t row = blockIdx.x, b = row / a.Hq, h = row - b * a.Hq, tid = threadIdx.x, lane = tid & 63u;
    const uint32_t per = a.D / 4, part = tid / per, d = (tid - part * per) * 4;
    const uint2 parts = *reinterpret_cast<const uint2*>(a.parts + 2 * b);
    // the only sequence's parts begin at 0: they can be requested before their number is known, up to what there is room for
    const uint32_t first = a.B == 1 ? 0u : parts.x, room = a.B == 1 ? a.shares : parts.y;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)first * a.Hq + h;
    const float* po = a.part_o + ((size_t)first * a.Hq + h) * a.D + d;
    const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
    // everything that a sequence's even portion of the parts needs is requested at once
    constexpr uint32_t kAhead = 4;
    floatx4 ahead[kAhead];
    float peak[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t s = part + i * groups;
        const bool there = part < groups && s < room;
        ahead[i] = there ? *reinterpret_cast<const floatx4*>(po + (size_t)s * a.Hq * a.D) : floatx4{0.f, 0.f, 0.f, 0.f};
        peak[i] = there ? ml[(size_t)s * a.Hq].x : -INFINITY;
    }
    // every wave finds the maximum and the sum for itself
    float2 own = lane < room ? ml[(size_t)lane * a.Hq] : make_float2(-INFINITY, 0.f);
    const uint32_t n = parts.y;
    if (n == 1) return;                      // the result is there
    if (lane >= n) own = make_float2(-INFINITY, 0.f);
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (part + i * groups >= n) peak[i] = -INFINITY;
    float top = fmaxf(own.x, sink);
    for (uint32_t s = lane + 64; s < n; s += 64) top = fmaxf(top, ml[(size_t)s * a.Hq].x);
    top = fmaxf(top, dpp_f<0xB1>(top));
    top = fmaxf(top, dpp_f<0x4E>(top));
    top = fmaxf(top, dpp_f<0x141>(top));
    top = rows_max(fmaxf(top, dpp_f<0x140>(top)));
    const float ref = top == -INFINITY ? 0.f : top;
    float total = __builtin_amdgcn_exp2f(own.x - ref) * own.y;
    for (uint32_t s = lane + 64; s < n; s += 64) {
        const float2 v = ml[(size_t)s * a.Hq];
        total += __builtin_amdgcn_exp2f(v.x - ref) * v.y;
    }
    total = rows_sum(group_sum<16>(total));
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    if (part < groups) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
            if (part + i * groups < n) sum += part_weight(peak[i] - ref) * ahead[i];
        for (uint32_t s = part + kAhead * groups; s < n; s += groups)
            sum += part_weight(ml[(size_t)s * a.Hq].x - ref) * *reinterpret_cast<const floatx4*>(po + (size_t)s * a.Hq * a.D);
        if (groups > 1) *reinterpret_cast<floatx4*>(sums + part * a.D + d) = sum;
    }
    if (groups > 1) __syncthreads();
    if (part != 0) return;
    for (uint32_t p = 1; p < groups; ++p) sum += *reinterpret_cast<const floatx4*>(sums + p * a.D + d);
    const float inv = 1.0f / (total + __builtin_amdgcn_exp2f(sink - ref));
    const float y[4] = {divided(sum[0], total, inv), divided(sum[1], total, inv), divided(sum[2], total, inv), divided(sum[3], total, inv)};
    store_rows(a, (size_t)row * a.D + d, y, true);
}

// Short sequences take a workgroup each.  Otherwise the tiles are shared equally by as many workgroups as stream the cache fastest: 512, two for each CU; three where
// heads are narrow, one where they are wide.  us by workgroups (256, 512, 768, 1024): 64 x 8192 tokens of 8 heads of 128, fp16 318, 321, 330, 328, Q8_0 201, 175, 183, 182;
// one Q8_0 sequence of 131071 57, 52, 56, 58; 64 ragged ones of up to 6001 with heads of 64 72, 53, 49, 49; 16 fp16 ones of 16384 with 2 heads of 256 89 (256), 97 (512).
// A share is two tiles a wave at least, but one where that leaves most CUs idle (one Q8_0 sequence of 2000: 11.1 -> 9.8 us; of 8000: 11.9, 12.8).
// The figures are of fp16 for wide heads, which one workgroup fills a CU with; Q8_0's, of which two fit, have not been measured with more than one.  Shares are rounded up, so that
// with a number of heads that does not divide these there are a few workgroups more, which wait for a place: 16384 fp16 tokens of 3, 5 and 6 heads of 256 4.6, 4.4 and 4.9 TB/s where
// 2, 4 and 8 reach 6.2 to 6.3, Q8_0 3.8 to 3.9 where they reach 5.5.
struct Plan {
    uint32_t shares;         // 0: a workgroup for each sequence and group of heads
    uint64_t ws_bytes;
};
constexpr uint32_t kDirectTiles = 4 * kWaves;
static Plan plan_of(uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t max_len, uint32_t window) {
    const uint32_t span = window && window < max_len ? window : max_len;
    const uint64_t tiles = window && window < max_len ? span / kTile + 2 : (span + (uint64_t)kTile - 1) / kTile, all = B * tiles;   // a window may begin within a tile
    const uint64_t groups = (uint64_t)Hkv * ((Hq / Hkv + 15) / 16);
    if (tiles <= kDirectTiles) return {0, 0};
    auto up = [](uint64_t x, uint64_t y) { return (x + y - 1) / y; };
    uint64_t most = up(all, kLeastShare);
    if (most * groups > 128) most = up(all, 2 * kLeastShare) > up(128, groups) ? up(all, 2 * kLeastShare) : up(128, groups);
    uint64_t shares = up(D > 128 ? 256 : D > 64 ? 512 : 768, groups);
    if (shares > most) shares = most;
    return {(uint32_t)shares, (shares + B) * Hq * (D + 2) * 4 + (uint64_t)B * 8};
}

template <bool Q8, int DP, int NBLK, bool FULL>
static int launch_form(mx_stream_t s, const AttnArgs& a, dim3 grid, uint32_t heads) {
    static LdsLimit limit;
    // keys, their scales and wide heads' queries; behind them the waves' sums, in the same place
    constexpr uint32_t keys = kWaves * kTile * (Q8 ? DP + 4 * NBLK : 2 * DP) + (DP > 128 ? DP * 32 : 0), most = kWaves * (32 + 16 * (DP + 4)) * 4;
    const uint32_t sums = kWaves * (32 + heads * (DP + 4)) * 4, lds = keys > sums ? keys : sums;
    if (lds > kLdsDefaultLimit)
        if (int rc = raise_lds_limit(reinterpret_cast<const void*>(attn_decode_kernel<Q8, DP, NBLK, FULL>), limit, keys > most ? keys : most)) return rc;
    hipLaunchKernelGGL((attn_decode_kernel<Q8, DP, NBLK, FULL>), grid, dim3(kWaves * 64), lds, as_stream(s), a);
    return launch_status();
}
static int launch_attn(mx_stream_t s, const AttnArgs& a, bool q8, dim3 grid, uint32_t heads) {
    if (q8) switch (a.D / 32) {
        case 1: return launch_form<true, 64, 1, false>(s, a, grid, heads);
        case 2: return launch_form<true, 64, 2, true>(s, a, grid, heads);
        case 3: return launch_form<true, 128, 3, false>(s, a, grid, heads);
        case 4: return launch_form<true, 128, 4, true>(s, a, grid, heads);
        case 5: return launch_form<true, 256, 5, false>(s, a, grid, heads);
        case 6: return launch_form<true, 256, 6, false>(s, a, grid, heads);
        case 7: return launch_form<true, 256, 7, false>(s, a, grid, heads);
        default: return launch_form<true, 256, 8, true>(s, a, grid, heads);
    }
    if (a.D == 64) return launch_form<false, 64, 2, true>(s, a, grid, heads);
    if (a.D < 64) return launch_form<false, 64, 2, false>(s, a, grid, heads);
    if (a.D == 128) return launch_form<false, 128, 4, true>(s, a, grid, heads);
    if (a.D < 128) return launch_form<false, 128, 4, false>(s, a, grid, heads);
    if (a.D == 256) return launch_form<false, 256, 8, true>(s, a, grid, heads);
    return launch_form<false, 256, 8, false>(s, a, grid, heads);
}

static int attn_decode(mx_stream_t s, bool q8, const uint16_t* q, uint64_t q_stride, const void* k, const uint16_t* k_d, const void* v, const uint16_t* v_d,
                       const int32_t* page_table, uint32_t max_pages, const int32_t* seq_lens, const float* sinks, uint16_t* out, void* out_q8, uint32_t B,
                       uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size, uint32_t max_len, uint32_t window, float scale, void* ws,
                       uint64_t ws_bytes) {
    MX_REQUIRE_PTR(q); MX_REQUIRE_PTR(k); MX_REQUIRE_PTR(v); MX_REQUIRE_PTR(page_table); MX_REQUIRE_PTR(seq_lens); MX_REQUIRE_PTR(out);
    if (q8) { MX_REQUIRE_PTR(k_d); MX_REQUIRE_PTR(v_d); }
    MX_REQUIRE_SHAPE(B > 0 && B <= 65535 && Hkv > 0 && Hkv <= 65535 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0);
    MX_REQUIRE_SHAPE(D > 0 && D <= 256 && D % (q8 ? 32 : 16) == 0 && q_stride % 8 == 0 && q_stride >= (uint64_t)Hq * D);
    MX_REQUIRE_SHAPE(n_pages > 0 && page_size > 0 && page_size % 16 == 0 && (uint64_t)n_pages * page_size < (1ull << 31) && max_pages > 0);
    const uint64_t tiles = (uint64_t)max_pages * page_size / kTile + 1;
    MX_REQUIRE_SHAPE(B * (tiles < (1u << 26) ? tiles : 1u << 26) < (1ull << 31));   // tiles of all sequences, counted in 32 bits
    MX_REQUIRE_SHAPE(!out_q8 || (uint64_t)Hq * D % 32 == 0);
    MX_REQUIRE_ALIGN(q, 16); MX_REQUIRE_ALIGN(k, 16); MX_REQUIRE_ALIGN(v, 16); MX_REQUIRE_ALIGN(out, 16); MX_REQUIRE_ALIGN(out_q8, 8);
    MX_REQUIRE_ALIGN(page_table, 4); MX_REQUIRE_ALIGN(seq_lens, 4); MX_REQUIRE_ALIGN(sinks, 4);
    if (q8) { MX_REQUIRE_ALIGN(k_d, 16); MX_REQUIRE_ALIGN(v_d, 16); }
    const Plan p = plan_of(B, Hq, Hkv, D, max_len, window);
    if (p.shares) {
        MX_REQUIRE_PTR(ws);
        MX_REQUIRE_ALIGN(ws, 16);
        if (ws_bytes < p.ws_bytes) return MX_ERR_WORKSPACE;
    }
    AttnArgs a = {};
    a.q = reinterpret_cast<const half_t*>(q); a.q_stride = q_stride;
    a.k = k; a.v = v; a.k_d = reinterpret_cast<const half_t*>(k_d); a.v_d = reinterpret_cast<const half_t*>(v_d);
    a.table = page_table; a.lens = seq_lens; a.sinks = sinks;
    a.out = reinterpret_cast<half_t*>(out);
    a.out_q8 = D % 32 == 0 ? static_cast<uint8_t*>(out_q8) : nullptr;   // heads of half a block: the quantizer, after the rows
    if (p.shares) {
        const uint64_t rows = ((uint64_t)p.shares + B) * Hq;
        a.part_o = static_cast<float*>(ws);
        a.part_ml = a.part_o + rows * D;
        a.parts = reinterpret_cast<uint32_t*>(a.part_ml + rows * 2);
    }
    a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.max_pages = max_pages; a.n_pages = n_pages; a.page_size = page_size;
    a.page_shift = (page_size & (page_size - 1)) == 0 ? (uint32_t)__builtin_ctz(page_size) : 32u;
    a.window = window; a.shares = p.shares;
    a.scale = scale * kLog2e;
    const uint32_t G = Hq / Hkv, heads = G < 16 ? G : 16;
    const uint64_t groups = (uint64_t)Hkv * ((G + 15) / 16);
    MX_REQUIRE_SHAPE(groups <= 65535 && (uint64_t)B * Hq < (1ull << 31));
    // the join's groups of parts: four parts a thread where a sequence has its even portion of them; a launch holds fewer than 2^32 threads
    uint32_t join_groups = (p.shares / B + 4) / 4;
    if (join_groups > 512 / (D / 4)) join_groups = 512 / (D / 4);
    const uint32_t join_threads = (join_groups * (D / 4) + 63) / 64 * 64;
    MX_REQUIRE_SHAPE(!p.shares || (uint64_t)B * Hq * join_threads < (1ull << 32));
    if (int rc = launch_attn(s, a, q8, dim3(p.shares ? p.shares : B, (uint32_t)groups), heads)) return rc;
    if (p.shares) {
        hipLaunchKernelGGL(attn_join_kernel, dim3(B * Hq), dim3(join_threads), join_groups * D * 4, as_stream(s), a, join_groups);
        if (int rc = launch_status()) return rc;
    }
    return out_q8 && !a.out_q8 ? mx_quantize_q8_1(s, out, out_q8, (uint64_t)B * Hq * D) : MX_OK;
}

}  // namespace mxq

using namespace mxq;

extern "C" {

int mx_attn_decode_ws_bytes(uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t max_len, uint32_t window, uint64_t* bytes) {
    MX_REQUIRE_PTR(bytes);
    MX_REQUIRE_SHAPE(B > 0 && B <= 65535 && Hkv > 0 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0 && D > 0 && D <= 256 && D % 16 == 0);
    *bytes = plan_of(B, Hq, Hkv, D, max_len, window).ws_bytes;
    return MX_OK;
}

int mx_attn_decode_f16(mx_stream_t s, const uint16_t* q, uint64_t q_stride, const uint16_t* k_cache, const uint16_t* v_cache, const int32_t* page_table,
                       uint32_t max_pages, const int32_t* seq_lens, const float* sinks, uint16_t* out, void* out_q8, uint32_t B, uint32_t Hq, uint32_t Hkv,
                       uint32_t D, uint32_t n_pages, uint32_t page_size, uint32_t max_len, uint32_t window, float scale, void* ws, uint64_t ws_bytes) {
    return attn_decode(s, false, q, q_stride, k_cache, nullptr, v_cache, nullptr, page_table, max_pages, seq_lens, sinks, out, out_q8, B, Hq, Hkv, D, n_pages,
                       page_size, max_len, window, scale, ws, ws_bytes);
}
int mx_attn_decode_q8_0(mx_stream_t s, const uint16_t* q, uint64_t q_stride, const int8_t* k_qs, const uint16_t* k_d, const int8_t* v_qs, const uint16_t* v_d,
                        const int32_t* page_table, uint32_t max_pages, const int32_t* seq_lens, const float* sinks, uint16_t* out, void* out_q8, uint32_t B,
                        uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size, uint32_t max_len, uint32_t window, float scale, void* ws,
                        uint64_t ws_bytes) {
    return attn_decode(s, true, q, q_stride, k_qs, k_d, v_qs, v_d, page_table, max_pages, seq_lens, sinks, out, out_q8, B, Hq, Hkv, D, n_pages, page_size, max_len,
                       window, scale, ws, ws_bytes);
}

}  // extern "C"
