"""Where the Q4_0 cache's kernels, the attention over it, the residual's norm and the routing read and write: their source compiled for the CPU and run as a GPU runs it, over
buffers that end at an unmapped page (see test_host_kv_bounds.py), and their results compared with plain sums.  No GPU."""
import pytest

import test_host_kv_bounds as B

MORE = r"""
#include <cmath>
template <class T> static T __shfl(T v, int l) { return from_lane(v, 9, 64, l & 63); }
template <class T> static T __shfl_xor(T v, int m) { return from_lane(v, 9, 64, lane_id() ^ m); }
#define __builtin_amdgcn_mbcnt_lo(m, c) ((uint32_t)__builtin_popcount((m) & (lane_id() < 32 ? (1u << lane_id()) - 1u : 0xFFFFFFFFu)) + (c))
#define __builtin_amdgcn_mbcnt_hi(m, c) ((uint32_t)__builtin_popcount((m) & (lane_id() < 32 ? 0u : (1u << (lane_id() - 32)) - 1u)) + (c))
#define __builtin_amdgcn_inverse_ballot_w64(m) (((uint64_t)(m) >> lane_id() & 1ull) != 0)
static uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)((uint64_t)a * b >> 32); }
// sixteen lanes bring the halves of eight rows of 16 bytes; lane r gets byte r of each
template <class V> static V shim_tr8(V* p) {
    const int l = lane_id() & 15, first = now / 16 * 16;
    const uint8_t* mine = reinterpret_cast<const uint8_t*>(p);
    memcpy(slot[now], &mine, sizeof mine);
    rendezvous(10, 64);
    uint8_t got[8];
    for (int k = 0; k < 8; ++k) { const uint8_t* row; memcpy(&row, slot[first + 2 * k + (l >> 3)], sizeof row); got[k] = row[l & 7]; }
    V v;
    memcpy(&v, got, 8);
    rendezvous(10, 64);
    return v;
}
#define __builtin_amdgcn_ds_read_tr8_b64_v2i32 shim_tr8
static int shim_dpp_or_rotation(int old, int v, int ctrl, int row_mask, int bank_mask, bool bound) {
    if (ctrl > 0x120 && ctrl <= 0x12F) return from_lane(v, 3, 16, ((lane_id() & 15) - (ctrl - 0x120)) & 15);
    return shim_dpp(old, v, ctrl, row_mask, bank_mask, bound);
}
#undef __builtin_amdgcn_update_dpp
#define __builtin_amdgcn_update_dpp shim_dpp_or_rotation
"""

ATTENTION = r"""
template <int NB, int C, int W = kWaves> static void one(uint32_t Hkv, uint32_t G, uint32_t ps, uint32_t window, uint32_t shares, std::vector<int32_t> lens, float scale = 0.3f, float q_size = 1.f, int plant = 0) {
    const uint32_t D = 32 * NB, B = (uint32_t)lens.size(), Hq = Hkv * G;
    uint32_t most = 1, pages = 0;
    for (int32_t n : lens) { const uint32_t need = n > 0 ? (n + ps - 1) / ps : 0; most = std::max(most, need); pages += need; }
    if (pages == 0) pages = 1;
    snprintf(what, sizeof what, "attention, Q4_0 D=%u, %d column groups, Hkv=%u G=%u pages of %u, window %u, %u shares, %u sequences of %d.., scale %g, queries of %g, plant %d\n", D, C, Hkv, G, ps, window, shares, B, lens[0], scale, q_size, plant);
    const size_t values = (size_t)pages * Hkv * ps * D;
    Held q(2 * (size_t)B * Hq * D), k(values / 2), v(values / 2), kd(values / 16), vd(values / 16), table(4 * (size_t)B * most), len(4 * B), sinks(4 * Hq),
        out(2 * (size_t)B * Hq * D), q8((size_t)B * Hq * D / 32 * 40 + 8), ws((((size_t)shares + B) * Hq * (D + 2) * 4 + B * 8 + 15) / 16 * 16);
    fill(q.as<half_t>(), (size_t)B * Hq * D);
    for (size_t i = 0; i < q.n / 2; ++i) q.as<half_t>()[i] = (half_t)((float)q.as<half_t>()[i] * q_size);
    for (size_t i = 0; i < values / 2; ++i) { k.p[i] = (uint8_t)rnd(256); v.p[i] = (uint8_t)rnd(256); }
    for (size_t i = 0; i < values / 32; ++i) {
        kd.as<half_t>()[i] = (half_t)((0.05f + 0.0001f * rnd(999)) * (rnd(2) ? 1 : -1) / q_size);
        vd.as<half_t>()[i] = (half_t)((0.05f + 0.0001f * rnd(999)) * (rnd(2) ? 1 : -1));
    }
    uint32_t next = pages;
    for (uint32_t b = 0; b < B; ++b) {
        len.as<int32_t>()[b] = lens[b];
        for (uint32_t i = 0; i < most; ++i) table.as<int32_t>()[b * most + i] = lens[b] > 0 && i < (lens[b] + ps - 1) / ps ? (int32_t)--next : 2147483647;
    }
    auto row_at = [&](uint32_t b, uint32_t hk, uint32_t t) { return (((size_t)table.as<int32_t>()[b * most + t / ps]) * Hkv + hk) * ps + t % ps; };
    if (plant == 1)       // scales of very different size, growing and shrinking along a sequence
        for (size_t i = 0; i < values / 32; ++i) vd.as<half_t>()[i] = (half_t)((float)vd.as<half_t>()[i] * exp2f((float)rnd(24) - 12.f));
    if (plant == 2)       // no numbers behind the sequences' ends
        for (uint32_t b = 0; b < B; ++b)
            for (uint32_t t = std::max(0, lens[b]); t < (std::max(0, lens[b]) + ps - 1) / ps * ps; ++t)
                for (uint32_t hk = 0; hk < Hkv; ++hk)
                    for (uint32_t n = 0; n < NB; ++n) { kd.as<half_t>()[row_at(b, hk, t) * NB + n] = (half_t)NAN; vd.as<half_t>()[row_at(b, hk, t) * NB + n] = (half_t)(rnd(2) ? INFINITY : NAN); }
    std::vector<bool> bad(values / 32, false);
    if (plant == 3)       // blocks of values that are no numbers
        for (size_t i = 0; i < values / 32; i += 1 + rnd(40)) { vd.as<half_t>()[i] = (half_t)(rnd(2) ? NAN : rnd(2) ? INFINITY : -INFINITY); bad[i] = true; }
    for (uint32_t h = 0; h < Hq; ++h) sinks.as<float>()[h] = real();
    memset(out.p, 0xFF, out.n);
    AttnArgs a = {};
    a.q = q.as<half_t>(); a.q_stride = (uint64_t)Hq * D; a.k = k.p; a.v = v.p; a.k_d = kd.as<half_t>(); a.v_d = vd.as<half_t>();
    a.table = table.as<int32_t>(); a.lens = len.as<int32_t>(); a.sinks = sinks.as<float>(); a.out = out.as<half_t>(); a.out_q8 = q8.p;
    a.part_o = ws.as<float>(); a.part_ml = a.part_o + ((size_t)shares + B) * Hq * D; a.parts = reinterpret_cast<uint32_t*>(a.part_ml + ((size_t)shares + B) * Hq * 2);
    a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.max_pages = most; a.n_pages = pages; a.page_size = ps; a.window = window; a.shares = shares;
    a.page_shift = (ps & (ps - 1)) == 0 ? (uint32_t)__builtin_ctz(ps) : 32u;
    a.scale = scale * kLog2e;
    const uint32_t heads = std::min(G, 16u);
    const size_t tiles = W * (2 * 36 * 16 * (NB | 1) + kTile * (2 * NB + 1) * 2), sums = W * (32 + heads * (D + 4)) * 4;   // as the launch asks for
    run(W * 64, shares ? shares : B, Hkv * ((G + 15) / 16), std::max(tiles, sums), [&] { if (shares) attn_decode_q4_kernel<NB, C, W, true>(a); else attn_decode_q4_kernel<NB, C, W, false>(a); });
    if (shares) {
        uint32_t groups = std::min((shares / B + 4) / 4, 512 / (D / 4));
        run((groups * (D / 4) + 63) / 64 * 64, B * Hq, 1, groups * D * 4, [&] { attn_join_kernel(a, groups); });
    }
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t h = 0; h < Hq; ++h) {
            const uint32_t n = lens[b] > 0 ? lens[b] : 0, lo = window && n > window ? n - window : 0, hk = h / G;
            std::vector<double> x, sum(D, 0.0), size(D, 0.0);
            std::vector<bool> none(D, false);
            double top = sinks.as<float>()[h], total;
            auto value = [&](Held& p, Held& d, size_t row, uint32_t i) {
                const uint8_t byte = p.p[row * (D / 2) + i / 32 * 16 + i % 16];
                return ((i & 16 ? byte >> 4 : byte & 15) - 8) * (double)(float)d.as<half_t>()[row * NB + i / 32];
            };
            for (uint32_t t = lo; t < n; ++t) {
                double s = 0;
                for (uint32_t i = 0; i < D; ++i) s += (double)(float)q.as<half_t>()[((size_t)b * Hq + h) * D + i] * value(k, kd, row_at(b, hk, t), i);
                x.push_back(scale * s);
                top = std::max(top, x.back());
            }
            total = exp(sinks.as<float>()[h] - top);
            for (uint32_t t = lo; t < n; ++t) {
                const double p = exp(x[t - lo] - top);
                total += p;
                for (uint32_t i = 0; i < D; ++i) {
                    if (bad[row_at(b, hk, t) * NB + i / 32]) { none[i] = true; continue; }
                    sum[i] += p * value(v, vd, row_at(b, hk, t), i);
                    size[i] += p * 8 * fabs((double)(float)vd.as<half_t>()[row_at(b, hk, t) * NB + i / 32]);
                }
            }
            for (uint32_t i = 0; i < D; ++i) {
                const double want = n ? sum[i] / total : 0.0, got = (double)(float)out.as<half_t>()[((size_t)b * Hq + h) * D + i];
                if (none[i] ? !std::isnan(got) : !(fabs(got - want) <= 1e-6 + 1e-3 * fabs(want) + 3e-4 * size[i] / total)) {
                    char m[100]; snprintf(m, sizeof m, "element %u of head %u of sequence %u is %g, not %g: ", i, h, b, got, want); wrong(m);
                }
            }
        }
}
int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    CASES
    return 0;
}
"""

# lengths that end within a tile, at its end, at a page's end, in the last page of the cache; every width of head, short and in shares; other sizes of queries and scales; planes with no numbers
ATTENTION_CASES = {
    "32": "one<1, 1>(2, 2, 16, 0, 0, {1, 33, 0}); one<1, 1>(1, 17, 48, 33, 3, {250, 0, 0, 48, 96});",
    "64": """one<2, 2>(1, 8, 16, 0, 0, {16, 129}); one<2, 2>(2, 1, 48, 33, 3, {250, 0, 0, 48, 96}); one<2, 2>(1, 4, 16, 0, 0, {300}, -0.3f, 1e-4f); one<2, 1>(1, 9, 16, 0, 0, {100, 33});
             one<2, 2>(1, 2, 16, 7, 0, {40, 7}, 0.f);""",
    "96": "one<3, 4>(1, 2, 16, 0, 0, {31, 32}); one<3, 4>(1, 1, 32, 40, 2, {200}); one<3, 2>(1, 5, 16, 0, 0, {45}); one<3, 1>(1, 10, 16, 0, 0, {45});",
    "128": "one<4, 4>(1, 4, 64, 0, 0, {65}); one<4, 4>(1, 2, 16, 0, 3, {300, 1, 0, 128}); one<4, 1>(1, 16, 16, 0, 0, {47}, 0.1f, 30.f); one<4, 2>(1, 7, 16, 0, 2, {300, 64});",
    "wide": """one<5, 8>(1, 1, 16, 0, 0, {17}); one<6, 8>(1, 2, 16, 0, 0, {32}); one<7, 8>(1, 1, 48, 0, 2, {140}); one<8, 8>(1, 2, 16, 0, 2, {150, 0, 31}); one<8, 8>(1, 1, 32, 9, 0, {64});
               one<5, 4>(1, 3, 16, 0, 0, {40}); one<6, 2>(1, 6, 16, 0, 0, {70}); one<7, 4>(1, 4, 16, 0, 0, {33}); one<8, 4>(1, 4, 16, 0, 2, {150}); one<8, 2>(1, 8, 16, 0, 0, {50}); one<8, 1>(1, 9, 16, 0, 0, {40});
               one<5, 1>(1, 12, 16, 0, 0, {20}); one<7, 2>(1, 5, 16, 0, 0, {20});""",
    "scales": """one<2, 2>(1, 3, 16, 0, 0, {333, 5}, 0.3f, 1.f, 1); one<4, 4>(1, 2, 32, 0, 3, {400, 31}, 0.3f, 1.f, 1); one<2, 2>(2, 1, 48, 0, 0, {17, 100, 1}, 0.3f, 1.f, 2);
                 one<3, 4>(1, 1, 16, 20, 2, {333, 18}, 0.3f, 1.f, 2);""",
    "eight_waves": "one<4, 4, 8>(1, 3, 16, 0, 0, {300, 0, 5}); one<2, 2, 8>(2, 8, 48, 0, 0, {513}, 0.3f, 1.f, 2); one<8, 1, 8>(1, 17, 16, 290, 0, {333}); one<1, 1, 8>(1, 1, 32, 0, 0, {700}); one<8, 8, 8>(1, 1, 16, 0, 0, {270});",
    "shares": """one<1, 1>(1, 1, 16, 0, 5, {1, 70, 0, 33, 300, 2, 0, 0, 31, 32, 64, 200, 16}); one<1, 1>(1, 2, 16, 0, 3, {128, 128, 128}); one<1, 1>(1, 1, 16, 40, 4, {500, 20, 41, 70, 90, 300}); one<1, 1>(1, 1, 16, 0, 40, {1, 2, 3});
                 { std::vector<int32_t> many; for (int i = 0; i < 70; ++i) many.push_back(i % 9 == 4 ? 0 : 1 + i * 37 % 130); one<1, 1>(1, 1, 16, 0, 11, many); }""",
    "no_numbers": "one<2, 2>(1, 3, 16, 0, 0, {133, 5}, 0.3f, 1.f, 3); one<4, 4>(1, 2, 32, 0, 3, {300, 31}, 0.3f, 1.f, 3); one<4, 2>(1, 5, 32, 0, 0, {100}, 0.3f, 1.f, 3);",
}


def attention_source():
    return B.source("attn_decode.hip", "// ---------------------------------------------------------------- launches").replace("__attribute__((address_space(3)))", "").replace(
        'asm("" : "+s"(minus));', "")


@pytest.mark.parametrize("form", sorted(ATTENTION_CASES))
def test_attention(tmp_path, form):
    B.build_and_run(tmp_path, B.SHIM + MORE + attention_source() + B.CHECK + ATTENTION.replace("CASES", ATTENTION_CASES[form]))


CACHE = r"""
static void encode(const float* x, uint8_t* codes, half_t* d) {      // a block, in exact quotients
    uint32_t at = 0;
    for (uint32_t i = 1; i < 32; ++i) if (fabsf(x[i]) > fabsf(x[at])) at = i;
    const double m = x[at];
    *d = (half_t)(float)(m == 0 ? -0.0 : m / -8);
    for (uint32_t i = 0; i < 32; ++i) {
        const int c = m == 0 ? 8 : std::min(15, (int)floor((double)x[i] * -8 / m + 8.5));
        codes[i % 16] = (uint8_t)(i < 16 ? c : codes[i % 16] | c << 4);
    }
}
static void cache(uint32_t T, uint32_t Hkv, uint32_t D, uint32_t ps, bool prompt, int plant) {
    const uint32_t pages = (T + ps - 1) / ps + 1, ks = Hkv * D + 16;
    snprintf(what, sizeof what, "%s of %u tokens, %u heads of %u, pages of %u, plant %d\n", prompt ? "prompt" : "rows", T, Hkv, D, ps, plant);
    const size_t values = (size_t)pages * Hkv * ps * D;
    Held k(2 * ((size_t)(T - 1) * ks + Hkv * D)), v(2 * ((size_t)(T - 1) * ks + Hkv * D)), kc(values / 2), vc(values / 2), kd(values / 16), vd(values / 16), slots(4 * T);
    fill(k.as<half_t>(), k.n / 2); fill(v.as<half_t>(), v.n / 2);
    for (size_t i = 0; plant && i < v.n / 2; ++i) {
        half_t& e = v.as<half_t>()[i];
        if (plant == 1) e = (half_t)((float)((int)rnd(33) - 16) / 16.f);              // next to every second one a border between two codes, and many of the largest size
        if (plant == 2) e = __builtin_bit_cast(half_t, (uint16_t)(rnd(2) << 15 | rnd(rnd(2) ? 40 : 0x7C00)));   // all of fp16
        if (plant == 3) e = (half_t)0.f;
    }
    for (uint32_t t = 0; t < T; ++t) slots.as<int32_t>()[t] = t % 5 == 3 ? (t % 2 ? -1 : (int32_t)(pages * ps)) : (int32_t)(pages * ps - 1 - t);
    memset(kc.p, 0xA5, kc.n); memset(vc.p, 0xA5, vc.n); memset(kd.p, 0xA5, kd.n); memset(vd.p, 0xA5, vd.n);
    RowsArgs a = {};
    a.k = k.as<half_t>(); a.v = v.as<half_t>(); a.k_stride = a.v_stride = ks;
    a.k_cache = kc.p; a.v_cache = vc.p; a.k_d = kd.as<half_t>(); a.v_d = vd.as<half_t>(); a.slots = slots.as<int32_t>();
    a.Hkv = Hkv; a.chunks = D / 8; a.page_size = ps; a.n_slots = pages * ps; a.mscale = 1.0;
    a.heads_per_wg = kRowThreads / a.chunks;
    a.groups = (2 * Hkv + a.heads_per_wg - 1) / a.heads_per_wg;
    const uint32_t items = 2 * Hkv * (a.chunks / 2), turns = (items + kRowThreads - 1) / kRowThreads, threads = ((items + turns - 1) / turns + 63) / 64 * 64;   // as launched
    if (prompt) run(threads, T, 1, 0, [&] { prompt_kernel<false, kQ4, false>(a); });
    else run(kRowThreads, a.groups * T, 1, 0, [&] { rows_kernel<false, kQ4, false>(a); });
    std::vector<bool> written(values / 32, false);
    for (uint32_t t = 0; t < T; ++t)
        for (uint32_t h = 0; h < 2 * Hkv; ++h) {
            const uint32_t slot = (uint32_t)slots.as<int32_t>()[t];
            if (slot >= a.n_slots) continue;
            const bool is_v = h >= Hkv;
            const uint32_t hk = is_v ? h - Hkv : h;
            const half_t* row = (is_v ? a.v : a.k) + t * (size_t)ks + hk * D;
            const size_t r = ((size_t)(slot / ps) * Hkv + hk) * ps + slot % ps;
            for (uint32_t n = 0; n < D / 32; ++n) {
                float x[32];
                uint8_t codes[16];
                half_t d;
                for (uint32_t i = 0; i < 32; ++i) x[i] = (float)row[n * 32 + i];
                encode(x, codes, &d);
                if (memcmp(codes, (is_v ? vc : kc).p + r * (D / 2) + n * 16, 16)) wrong("other codes: ");
                if (memcmp(&d, (is_v ? a.v_d : a.k_d) + r * (D / 32) + n, 2)) wrong("another scale: ");
                written[r * (D / 32) + n] = true;
            }
        }
    for (size_t i = 0; i < values / 32; ++i) if (!written[i]) { if (kc.p[i * 16] != 0xA5 || vc.p[i * 16 + 15] != 0xA5 || kd.as<uint16_t>()[i] != 0xA5A5 || vd.as<uint16_t>()[i] != 0xA5A5) wrong("a slot of no token: "); }
}
static void read(uint32_t Hkv, uint32_t D, uint32_t ps, std::vector<int32_t> lens, int32_t spare) {
    const uint32_t B = (uint32_t)lens.size();
    uint32_t most = 1, pages = 0, total = 0;
    for (int32_t n : lens) { most = std::max(most, (n + ps - 1) / ps); pages += (n + ps - 1) / ps; total += n; }
    snprintf(what, sizeof what, "reading back, %u sequences, %u rows, %u heads of %u, pages of %u\n", B, total, Hkv, D, ps);
    const size_t values = (size_t)pages * Hkv * ps * D;
    Held k(values / 2), v(values / 2), kd(values / 16), vd(values / 16), table(4 * (size_t)B * most), rows(4 * (B + 1)), ko((size_t)(total + spare) * Hkv * D * 2), vo((size_t)(total + spare) * Hkv * D * 2);
    for (size_t i = 0; i < k.n; ++i) { k.p[i] = (uint8_t)rnd(256); v.p[i] = (uint8_t)rnd(256); }
    for (size_t i = 0; i < values / 32; ++i) { kd.as<half_t>()[i] = (half_t)(0.001f * rnd(9999)); vd.as<half_t>()[i] = (half_t)(-0.0371f * rnd(9999)); }
    memset(ko.p, 0xFF, ko.n); memset(vo.p, 0xFF, vo.n);
    int32_t at = 0, next = (int32_t)pages;
    for (uint32_t b = 0; b < B; ++b) {
        rows.as<int32_t>()[b] = at;
        at += lens[b];
        for (uint32_t i = 0; i < most; ++i) table.as<int32_t>()[b * most + i] = i < (lens[b] + ps - 1) / ps ? --next : -1;
    }
    rows.as<int32_t>()[B] = at;
    READ_LAUNCH
    for (uint32_t b = 0; b < B; ++b)
        for (int32_t t = 0; t < lens[b]; ++t)
            for (uint32_t i = 0; i < Hkv * D; ++i) {
                const size_t r = ((size_t)table.as<int32_t>()[b * most + t / ps] * Hkv + i / D) * ps + t % ps, dst = (size_t)(rows.as<int32_t>()[b] + t) * Hkv * D + i;
                const uint32_t e = i % D;
                for (int side = 0; side < 2; ++side) {
                    const uint8_t byte = (side ? v : k).p[r * (D / 2) + e / 32 * 16 + e % 16];
                    const half_t want = (half_t)((float)((e & 16 ? byte >> 4 : byte & 15) - 8) * (float)(side ? vd : kd).as<half_t>()[r * (D / 32) + e / 32]);
                    if ((float)want != (float)(side ? vo : ko).as<half_t>()[dst]) wrong(side ? "another value: " : "another key: ");
                }
            }
    for (size_t i = (size_t)total * Hkv * D; i < ko.n / 2; ++i) if (ko.as<uint16_t>()[i] != 0xFFFF || vo.as<uint16_t>()[i] != 0xFFFF) wrong("rows behind the last sequence: ");
}
int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    for (int plant = 0; plant < 4; ++plant) {
        cache(3, 2, 64, 16, false, plant); cache(2, 8, 128, 16, false, plant); cache(7, 1, 96, 48, false, plant); cache(5, 3, 32, 32, false, plant); cache(6, 1, 256, 16, false, plant);
        cache(9, 3, 64, 16, true, plant); cache(4, 2, 256, 48, true, plant); cache(5, 1, 128, 16, true, plant);
    }
    read(2, 64, 16, {0, 16, 1}, 0); read(1, 96, 16, {33, 2}, 0); read(2, 256, 64, {65, 0}, 2); read(9, 32, 16, {3, 3, 3, 20}, 0);
    std::vector<int32_t> many;
    for (int i = 0; i < 150; ++i) many.push_back(i % 7 == 3 ? 0 : i % 5);
    read(1, 32, 16, many, 5);
    return 0;
}
"""

READ_LAUNCH = r"""run(256, (total + spare) / 16 + B, (2 * Hkv * 16 * (D / 8) + 256 * kReadPieces - 1) / (256 * kReadPieces), 0, [&] {
        kv_read_kernel<kQ4, false>(k.p, kd.as<half_t>(), v.p, vd.as<half_t>(), table.as<int32_t>(), most, rows.as<int32_t>(), ko.as<half_t>(), vo.as<half_t>(), total + spare, B, Hkv, D / 8, pages, ps);
    });"""


def test_rows_and_cache(tmp_path):
    source = B.source("kv_cache.hip", "// ---------------------------------------------------------------- argument checks")
    source = source.replace("constexpr uint32_t kPromptTokens", "#if 0\nconstexpr uint32_t kPromptTokens").replace("// Reading back: a workgroup", "#endif\n// Reading back: a workgroup")
    B.build_and_run(tmp_path, B.SHIM + MORE + source + B.CHECK + CACHE.replace("READ_LAUNCH", READ_LAUNCH))


NORM = r"""
enum { ROWS, FAR, SHORT };
template <int KIND, int P, bool HALVES> static void norm(uint32_t T, uint32_t hidden, bool in_place, bool want_y) {
    snprintf(what, sizeof what, "norm of %u rows of %u, form %d %d, %s, %s, %s\n", T, hidden, KIND, P, HALVES ? "halves" : "blocks", in_place ? "in place" : "apart", want_y ? "rows" : "no rows");
    const size_t n = (size_t)T * hidden, size = HALVES ? 48 : 40;
    Held x(2 * n), res(2 * n), w(4 * hidden), total(2 * n), y(2 * n), q8(n / 32 * size);
    fill(x.as<half_t>(), n); fill(res.as<half_t>(), n);
    for (uint32_t i = 0; i < hidden; ++i) w.as<float>()[i] = real();
    std::vector<half_t> sum(n);
    for (size_t i = 0; i < n; ++i) sum[i] = (half_t)((float)x.as<half_t>()[i] + (float)res.as<half_t>()[i]);
    half_t* const to = in_place ? res.as<half_t>() : total.as<half_t>();
    const SumArgs a = {x.as<half_t>(), res.as<half_t>(), w.as<float>(), to, want_y ? y.as<half_t>() : nullptr, q8.p, T, hidden, 1e-5f};
    const uint32_t passes = (hidden + kSumThreads * 8 - 1) / (kSumThreads * 8);
    if constexpr (KIND == ROWS) run(kSumThreads * std::min(passes, (uint32_t)P), T, 1, passes * kSumThreads * 16, [&] { add_norm_kernel<HALVES, false>(a); });
    if constexpr (KIND == FAR) run(kSumThreads * std::min(passes, (uint32_t)P), T, 1, 0, [&] { add_norm_kernel<HALVES, true>(a); });
    if constexpr (KIND == SHORT) run(256, (T + 256 / P - 1) / (256 / P), 1, 0, [&] { add_norm_short_kernel<P, HALVES>(a); });
    for (uint32_t t = 0; t < T; ++t) {
        double sq = 0;
        for (uint32_t i = 0; i < hidden; ++i) sq += (double)(float)sum[t * hidden + i] * (double)(float)sum[t * hidden + i];
        const double r = 1.0 / sqrt(sq / hidden + 1e-5);
        for (uint32_t i = 0; i < hidden; ++i) {
            const size_t at = (size_t)t * hidden + i;
            if (memcmp(&sum[at], to + at, 2)) wrong("another sum: ");
            const double want = (double)(float)sum[at] * r * w.as<float>()[i];
            if (want_y && !(fabs((double)(float)y.as<half_t>()[at] - want) <= 1e-3 * fabs(want) + 1e-7)) wrong("another norm: ");
            const uint8_t* blk = q8.p + at / 32 * size;
            const float d = *reinterpret_cast<const float*>(blk);
            if (!(fabs((double)d * (int8_t)blk[size - 32 + i % 32] - want) <= 0.51 * d + 1e-3 * fabs(want))) wrong("another code: ");
        }
    }
}
int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    // four passes at a time here, where a GPU has eight
    norm<ROWS, 4, true>(2, 992, true, true); norm<ROWS, 4, false>(1, 1024, false, false); norm<ROWS, 4, false>(2, 1056, true, true); norm<ROWS, 4, true>(1, 2880, false, false);
    norm<ROWS, 4, false>(2, 4096, false, true); norm<ROWS, 4, true>(1, 8224, true, true); norm<FAR, 4, false>(2, 4128, false, true); norm<FAR, 4, true>(1, 33024, true, false);
    norm<SHORT, 16, false>(35, 32, false, true); norm<SHORT, 16, true>(16, 96, true, true); norm<SHORT, 16, false>(1, 128, false, false); norm<SHORT, 32, true>(9, 160, true, true);
    norm<SHORT, 32, false>(3, 256, false, true); norm<SHORT, 64, true>(5, 288, false, true); norm<SHORT, 64, false>(4, 512, true, false);
    return 0;
}
"""


def between(name, begin, end):
    text = open(B.os.path.join(B.CSRC, name)).read()
    assert text.count(begin) == 1 and text.count(end) == 1
    return text[text.index(begin):text.index(end)]


def with_header(text):
    head = B.source("attn_decode.hip", "constexpr float kLog2e")     # the device header in place, and nothing else
    return head + "namespace mxq {\n" + text + "}  // namespace mxq\n"


def test_norm(tmp_path):
    kernel = between("producers.hip", "typedef _Float16 half8", "// y = half(silu(gate) * up) (swiglu,").replace('asm("" : "+v"(bits));', "").replace(
        "extern __shared__ char sums[];", "char* const sums = shim_lds;")
    B.build_and_run(tmp_path, B.SHIM + MORE + "static float rsqrtf(float x) { return 1.f / sqrtf(x); }\n" + with_header(kernel) + B.CHECK + NORM)


ROUTE = r"""
enum { SIGMOID = MX_ROUTE_SIGMOID, RENORM = MX_ROUTE_RENORM, TOP2 = MX_ROUTE_TOP2, F32 = MX_ROUTE_F32 };
template <int NJ> static void route(uint32_t T, uint32_t E, uint32_t K, uint32_t groups, uint32_t kept, uint32_t flags, bool with_bias, int plant) {
    snprintf(what, sizeof what, "routing of %u tokens to %u of %u experts, %u of %u groups, flags %u, %s, plant %d\n", T, K, E, kept, groups, flags, with_bias ? "bias" : "no bias", plant);
    Held logits((size_t)T * E * (flags & F32 ? 4 : 2)), bias(4 * E), idx(4 * T * K), w(2 * T * K);
    auto logit = [&](size_t i) { return flags & F32 ? logits.as<float>()[i] : (float)logits.as<half_t>()[i]; };
    for (size_t i = 0; i < (size_t)T * E; ++i) {
        float v = plant == 1 ? (float)rnd(3) : real() * 2;                                          // 1: almost all equal
        if (plant == 2 && rnd(4) == 0) v = rnd(3) ? -INFINITY : NAN;
        if (plant == 3) v = -INFINITY;
        if (flags & F32) logits.as<float>()[i] = v; else logits.as<half_t>()[i] = (half_t)v;
    }
    for (uint32_t e = 0; e < E; ++e) bias.as<float>()[e] = plant == 1 ? 0.f : real() * 0.1f;
    const uint32_t size = E / groups;
    RouteArgs a = {logits.p, with_bias ? bias.as<float>() : nullptr, idx.as<int32_t>(), w.as<half_t>(), T, E, K, groups, size, size > 1 ? 0xFFFFFFFFu / size + 1u : 0u, kept, 1, flags, 2.5f, E % NJ == 0};
    while (a.lanes * 2 * groups <= 64) a.lanes *= 2;
    memset(idx.p, 0xFF, idx.n);
    run(256, (T + 3) / 4, 1, 0, [&] { route_kernel<NJ>(a); });
    for (uint32_t t = 0; t < T; ++t) {
        std::vector<double> s(E), c(E);
        double top = -INFINITY, sum = 0;
        for (uint32_t e = 0; e < E; ++e) top = std::fmax(top, logit((size_t)t * E + e));
        for (uint32_t e = 0; e < E; ++e) {
            const double v = logit((size_t)t * E + e);
            s[e] = flags & SIGMOID ? 1 / (1 + exp(-v)) : v == -INFINITY ? 0 : exp(v - top);
            sum += s[e];
        }
        for (uint32_t e = 0; e < E; ++e) {
            if (!(flags & SIGMOID)) s[e] = sum == 0 ? 0 : s[e] / sum;
            c[e] = s[e] + (with_bias ? (double)bias.as<float>()[e] : 0.0);
        }
        auto before = [](double x, double y) { return std::isnan(y) ? !std::isnan(x) : x > y; };     // x in front of y whatever their places
        std::vector<uint32_t> g(groups), all;
        std::vector<double> worth(groups);
        for (uint32_t i = 0; i < groups; ++i) {
            g[i] = i;
            std::vector<double> m(c.begin() + i * size, c.begin() + (i + 1) * size);
            std::stable_sort(m.begin(), m.end(), before);
            worth[i] = flags & TOP2 && size > 1 ? m[0] + m[1] : m[0];
        }
        std::stable_sort(g.begin(), g.end(), [&](uint32_t x, uint32_t y) { return before(worth[x], worth[y]); });
        for (uint32_t e = 0; e < E; ++e) if (groups == 1 || std::find(g.begin(), g.begin() + kept, e / size) != g.begin() + kept) all.push_back(e);
        std::stable_sort(all.begin(), all.end(), [&](uint32_t x, uint32_t y) { return before(c[x], c[y]); });
        all.resize(K);
        std::sort(all.begin(), all.end());
        double of = 1;
        if (flags & RENORM) { of = 1e-20; for (uint32_t e : all) of += s[e]; }
        for (uint32_t k = 0; k < K; ++k) {
            if (idx.as<int32_t>()[t * K + k] != (int32_t)all[k]) wrong("another expert: ");
            const double want = 2.5 * s[all[k]] / of, got = (double)(float)w.as<half_t>()[t * K + k];
            if (std::isnan(want) ? !std::isnan(got) : !(fabs(got - want) <= 5e-4 * want + 1e-7)) wrong("another weight: ");
        }
    }
}
int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    for (int plant = 0; plant < 4; ++plant)
        for (uint32_t flags = 0; flags < 16; flags += 1 + (plant > 0)) {
            const bool bias = (flags >> 1 ^ plant) & 1;
            route<1>(5, 60, 7, 1, 1, flags, bias, plant); route<1>(1, 1, 1, 1, 1, flags, bias, plant); route<1>(4, 64, 64, 64, 64, flags, bias, plant); route<1>(3, 60, 3, 3, 2, flags, bias, plant);
            route<2>(2, 128, 8, 16, 5, flags, bias, plant); route<4>(3, 256, 8, 8, 4, flags, bias, plant); route<4>(2, 160, 6, 5, 1, flags, bias, plant); route<8>(2, 512, 16, 2, 1, flags, bias, plant);
            route<16>(1, 1000, 50, 40, 3, flags, bias, plant); route<16>(1, 1024, 64, 64, 64, flags, bias, plant);
        }
    return 0;
}
"""


def test_route(tmp_path):
    kernel = between("routing.hip", "__device__ __forceinline__ float wave_max_f", "// One wave per token, lane l holds the experts l, l + 64") + between(
        "routing.hip", "// A 64-bit number as an unsigned one", "// ---------------------------------------------------------------- packing")
    flags = "enum { MX_ROUTE_SIGMOID = 1, MX_ROUTE_RENORM = 2, MX_ROUTE_TOP2 = 4, MX_ROUTE_F32 = 8 };\n"
    B.build_and_run(tmp_path, B.SHIM + MORE + with_header(flags + kernel) + B.CHECK + ROUTE)
