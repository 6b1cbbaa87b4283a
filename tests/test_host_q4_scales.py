"""Scales of a Q4_0 cache that are no numbers: an infinite one makes its block NaN as a NaN does, for attention (keys: all of the heads that read it) and when it is read back.
The kernels' source compiled for the CPU and run as in test_host_q4_bounds.py.  No GPU."""
import test_host_kv_bounds as B
import test_host_q4_bounds as Q


def replaced(text, old, new):
    assert text.count(old) == 1, old
    return text.replace(old, new)


# plant 4: infinite scales among the keys' live blocks, of either sign; whole heads are NaN where their tokens have one
KEYS = replaced(replaced(Q.ATTENTION, "    for (uint32_t h = 0; h < Hq; ++h) sinks", """    if (plant == 4)
        for (size_t i = rnd(90); i < values / 32; i += 1 + rnd(90)) kd.as<half_t>()[i] = (half_t)(rnd(2) ? INFINITY : -INFINITY);
    for (uint32_t h = 0; h < Hq; ++h) sinks"""), "            total = exp(sinks.as<float>()[h] - top);", """            for (uint32_t t = lo; plant == 4 && t < n; ++t)
                for (uint32_t i = 0; i < NB; ++i) if (std::isinf((float)kd.as<half_t>()[row_at(b, hk, t) * NB + i])) none.assign(D, true);
            total = exp(sinks.as<float>()[h] - top);""")

KEY_CASES = """one<2, 2>(1, 3, 16, 0, 0, {33, 5, 1, 0, 16}, 0.3f, 1.f, 4); one<4, 4>(2, 2, 32, 0, 3, {100, 31, 7, 0, 64}, 0.3f, 1.f, 4); one<4, 2>(1, 5, 32, 0, 0, {20}, -0.3f, 1.f, 4);
    one<1, 1>(1, 1, 16, 7, 0, {40, 20, 30, 8, 9, 10}, 0.3f, 1.f, 4); one<3, 4>(1, 1, 16, 20, 2, {133, 18}, 0.3f, 1.f, 4); one<8, 8>(1, 2, 16, 0, 0, {9, 3}, 0.3f, 1.f, 4);
    one<5, 8>(2, 1, 16, 0, 0, {17, 2}, 0.3f, 1.f, 4); one<4, 4, 8>(1, 3, 16, 0, 0, {30, 0, 5}, 0.f, 1.f, 4);"""


def test_keys(tmp_path):
    B.build_and_run(tmp_path, B.SHIM + Q.MORE + Q.attention_source() + B.CHECK + KEYS.replace("CASES", KEY_CASES))


READ = replaced(replaced(replaced(Q.CACHE, "    memset(ko.p, 0xFF, ko.n);", """    for (size_t i = 0; i < values / 32; i += 1 + rnd(5)) (rnd(2) ? kd : vd).as<half_t>()[i] = (half_t)(rnd(3) ? rnd(2) ? INFINITY : -INFINITY : rnd(2) ? NAN : 65504.f);
    memset(ko.p, 0xFF, ko.n);"""), "                    if ((float)want !=", """                    const float d = (float)(side ? vd : kd).as<half_t>()[r * (D / 32) + e / 32], got = (float)(side ? vo : ko).as<half_t>()[dst];
                    if (std::isnan(d) || std::isinf(d)) { if (!std::isnan(got)) wrong("a number of a block that has none: "); continue; }
                    if ((float)want !="""), "static void cache(uint32_t T", "[[maybe_unused]] static void cache(uint32_t T")


def test_reading_back(tmp_path):
    source = B.source("kv_cache.hip", "// ---------------------------------------------------------------- argument checks")
    source = source.replace("constexpr uint32_t kPromptTokens", "#if 0\nconstexpr uint32_t kPromptTokens").replace("// Reading back: a workgroup", "#endif\n// Reading back: a workgroup")
    B.build_and_run(tmp_path, B.SHIM + Q.MORE + source + B.CHECK + READ.replace("READ_LAUNCH", Q.READ_LAUNCH))
