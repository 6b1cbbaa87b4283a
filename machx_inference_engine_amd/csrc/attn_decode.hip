// attn_decode.hip — attention of one new token over a paged key-value cache (fp16 or Q8_0 planes).
#include "mxq_device.h"
#include "mxq_host.h"

namespace mxq {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    const half_t* q;
    uint64_t q_stride;
    const void *k, *v;              // fp16, or int8
    const half_t *k_d, *v_d;        // Q8_0 scales
    const int32_t *table, *lens;
    const float* sinks;
    half_t* out;
    uint8_t* out_q8;
    uint32_t Hq, Hkv, D, max_pages, n_pages, page_size, window;
    float scale;
};

// One workgroup of four waves for each (sequence, query head); wave w takes the tokens w, w + 4, ...; the lanes of a wave share the elements of a row.
template <bool Q8>
__global__ __launch_bounds__(256) void attn_decode_kernel(AttnArgs a) {
    __shared__ float ms[4], ls[4], os[4][256];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, h = blockIdx.x, b = blockIdx.y, hk = h / (a.Hq / a.Hkv);
    const uint64_t capacity = (uint64_t)a.max_pages * a.page_size;
    const int32_t raw = a.lens[b];
    const uint32_t len = raw <= 0 ? 0u : (uint32_t)min((uint64_t)raw, capacity), start = a.window && len > a.window ? len - a.window : 0u;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t d = lane + 64 * i;
        q[i] = d < a.D ? (float)a.q[b * a.q_stride + (size_t)h * a.D + d] * (a.scale * kLog2e) : 0.f;
    }
    for (uint32_t t = start + wave; t < len; t += 4) {
        const uint32_t col = t / a.page_size, page = (uint32_t)a.table[(size_t)b * a.max_pages + col];
        if (page >= a.n_pages) continue;
        const size_t row = ((size_t)page * a.Hkv + hk) * a.page_size + (t - col * a.page_size);
        float x = 0.f, v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t d = lane + 64 * i;
            v[i] = 0.f;
            if (d >= a.D) continue;
            float k;
            if (Q8) {
                k = (float)static_cast<const int8_t*>(a.k)[row * a.D + d] * (float)a.k_d[row * (a.D / 32) + d / 32];
                v[i] = (float)static_cast<const int8_t*>(a.v)[row * a.D + d] * (float)a.v_d[row * (a.D / 32) + d / 32];
            } else {
                k = (float)static_cast<const half_t*>(a.k)[row * a.D + d];
                v[i] = (float)static_cast<const half_t*>(a.v)[row * a.D + d];
            }
            x += q[i] * k;
        }
        x = __shfl(group_sum<64>(x), 63);
        const float top = fmaxf(m, x), ref = top == -INFINITY ? 0.f : top, keep = exp2f(m - ref), p = exp2f(x - ref);
        m = top;
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * keep + p * v[i];
    }
    if (lane == 0) {
        ms[wave] = m;
        ls[wave] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) os[wave][lane + 64 * i] = o[i];
    __syncthreads();
    const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
    float top = sink;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ms[w]);
    if (top == -INFINITY) top = 0.f;
    float total = exp2f(sink - top), sum = 0.f;
    const uint32_t d = threadIdx.x;
    for (int w = 0; w < 4; ++w) {
        const float f = exp2f(ms[w] - top);
        total += f * ls[w];
        sum += f * os[w][d];
    }
    if (d < a.D) a.out[((size_t)b * a.Hq + h) * a.D + d] = f32_to_f16_rne(total == 0.f ? 0.f : sum / total);
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
    MX_REQUIRE_SHAPE(!out_q8 || (uint64_t)Hq * D % 32 == 0);
    MX_REQUIRE_ALIGN(q, 16); MX_REQUIRE_ALIGN(k, 16); MX_REQUIRE_ALIGN(v, 16); MX_REQUIRE_ALIGN(out, 16); MX_REQUIRE_ALIGN(out_q8, 8);
    MX_REQUIRE_ALIGN(page_table, 4); MX_REQUIRE_ALIGN(seq_lens, 4); MX_REQUIRE_ALIGN(sinks, 4);
    if (q8) { MX_REQUIRE_ALIGN(k_d, 2); MX_REQUIRE_ALIGN(v_d, 2); }
    AttnArgs a = {reinterpret_cast<const half_t*>(q), q_stride, k, v, reinterpret_cast<const half_t*>(k_d), reinterpret_cast<const half_t*>(v_d), page_table,
                  seq_lens, sinks, reinterpret_cast<half_t*>(out), static_cast<uint8_t*>(out_q8), Hq, Hkv, D, max_pages, n_pages, page_size, window, scale};
    (void)max_len; (void)ws; (void)ws_bytes;
    if (q8) hipLaunchKernelGGL((attn_decode_kernel<true>), dim3(Hq, B), dim3(256), 0, as_stream(s), a);
    else hipLaunchKernelGGL((attn_decode_kernel<false>), dim3(Hq, B), dim3(256), 0, as_stream(s), a);
    if (int rc = launch_status()) return rc;
    return out_q8 ? mx_quantize_q8_1(s, out, out_q8, (uint64_t)B * Hq * D) : MX_OK;
}

}  // namespace mxq

using namespace mxq;

extern "C" {

int mx_attn_decode_ws_bytes(uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t max_len, uint32_t window, uint64_t* bytes) {
    MX_REQUIRE_PTR(bytes);
    MX_REQUIRE_SHAPE(B > 0 && B <= 65535 && Hkv > 0 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0 && D > 0 && D <= 256 && D % 16 == 0);
    (void)max_len; (void)window;
    *bytes = 0;
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
