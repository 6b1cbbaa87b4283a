"""The one-token attention's kernels over values at the edge of fp16 and such that are no numbers, run on the CPU as a GPU runs them and compared with sums in 64 bits.  No GPU."""
import pytest

import test_host_kv_bounds as B

FILLED, CHECKED = "uint32_t next = pages;", "if (!(fabs(got - want)"


def run(tmp_path, plant, cases):
    """`plant` changes the planes between their filling and the launch."""
    program = B.ATTENTION.replace("CASES", cases)
    assert program.count(FILLED) == 1 and program.count(CHECKED) == 1
    program = program.replace(FILLED, plant + FILLED).replace(CHECKED, "if (got == want || (std::isnan(got) && std::isnan(want))) continue; " + CHECKED)
    B.build_and_run(tmp_path, B.SHIM + "#include <cmath>\n" + B.source("attn_decode.hip", "// Short sequences take a workgroup each.") + B.CHECK + program)


# infinities of one sign in the first elements of a head, of either in some behind them, NaN in others; the last tokens of a page among them, masked or not
PLANT = """for (size_t row = 0; row < values / D; row += 1 + rnd(60)) {
               const float inf = INFINITY, what[4] = {inf, -inf, rnd(2) ? inf : -inf, (float)NAN};
               for (uint32_t i = 0; i < 4; ++i) if (rnd(2)) v.as<half_t>()[row * D + i * 4 + rnd(2)] = (half_t)what[i];
           }
           """
# keys of 20 times the size: scores 100 and more apart, so that most weights, most waves' and parts' too, are zero in 32 bits
STEEP = "for (size_t i = 0; i < values; ++i) k.as<half_t>()[i] = (half_t)(20.f * (float)k.as<half_t>()[i]);\n"

CASES = [
    "one<false, 64, 2, true>(64, 2, 3, 16, 0, 0, {1, 16, 17, 0, 333}); one<false, 64, 2, false>(48, 2, 1, 32, 7, 0, {40}); one<false, 64, 2, true>(64, 1, 4, 16, 100, 3, {0, 300, 31, 0, 129, 1, 0});",
    "one<false, 128, 4, true>(128, 1, 4, 16, 0, 0, {31, 230}); one<false, 128, 4, false>(112, 1, 1, 64, 20, 2, {200, 65}); one<false, 128, 4, true>(128, 1, 17, 32, 0, 4, {700, 0, 64});",
    "one<false, 256, 8, true>(256, 1, 2, 16, 0, 0, {133}); one<false, 256, 8, false>(240, 1, 1, 48, 0, 2, {350, 47}); one<false, 256, 8, true>(256, 1, 3, 32, 50, 2, {160, 0, 97});"]


@pytest.mark.parametrize("steep", [False, True])
@pytest.mark.parametrize("cases", CASES, ids=["narrow", "128", "wide"])
def test_infinite_values(tmp_path, cases, steep):
    """An element is infinite where a token's value is, whatever that token's weight, and NaN where infinities of either sign or a NaN are."""
    run(tmp_path, PLANT + (STEEP if steep else ""), cases)


# fp16's largest number, 65504, is held as 127 times 516: 65532, which fp16 does not hold
LARGEST = """for (size_t i = 0; i < values / 32; i += 1 + rnd(5)) {
                 vd.as<half_t>()[i] = (half_t)516.f;
                 for (uint32_t e = 0; e < 32; ++e) v.as<int8_t>()[i * 32 + e] = (int8_t)(e % 7 ? (int)rnd(255) - 127 : rnd(2) ? 127 : -127);
             }
             """
# blocks as they are written of a NaN or an infinity: values of zero, a scale that is no number
NO_NUMBER = """for (size_t i = 0; i < values / 32; i += 1 + rnd(40)) {
                   vd.as<half_t>()[i] = rnd(2) ? (half_t)NAN : (half_t)INFINITY;
                   for (uint32_t e = 0; e < 32; ++e) v.as<int8_t>()[i * 32 + e] = 0;
               }
               """
Q8_CASES = [
    "one<true, 64, 1, false>(32, 2, 2, 16, 0, 0, {1, 33, 0}); one<true, 64, 2, true>(64, 1, 8, 16, 0, 0, {16, 129}); one<true, 64, 2, true>(64, 2, 1, 48, 33, 3, {250, 0, 0, 48, 96});",
    "one<true, 128, 3, false>(96, 1, 2, 16, 0, 0, {31, 32}); one<true, 128, 4, true>(128, 1, 2, 16, 0, 3, {300, 1, 0, 128});",
    "one<true, 256, 5, false>(160, 1, 1, 16, 0, 0, {17}); one<true, 256, 8, true>(256, 1, 2, 16, 0, 2, {150, 0, 31});"]


@pytest.mark.parametrize("plant", [LARGEST, NO_NUMBER], ids=["largest", "no_number"])
@pytest.mark.parametrize("cases", Q8_CASES, ids=["narrow", "128", "wide"])
def test_q8_0_values(tmp_path, cases, plant):
    """65504, stored as 65532, weighs as that; a block that holds no number is NaN wherever one of its tokens counts."""
    run(tmp_path, plant, cases)


def test_two_parts_hold_every_q8_0_value(tmp_path):
    """Every scale up to 516 (fp16's largest number, 65504, over 127) times every value: a first part that fp16 holds and an exact second one."""
    B.build_and_run(tmp_path, B.SHIM + B.source("attn_decode.hip", "// Short sequences take a workgroup each.") + B.CHECK + r"""
int main() {
    for (uint32_t bits = 0; bits <= 0x6008; ++bits) {
        const half_t d = __builtin_bit_cast(half_t, (uint16_t)bits);
        half8 all;
        for (int i = 0; i < 8; ++i) all[i] = d;
        const half_t most = at_most_511(all)[bits % 8];
        for (int q = -128; q < 128; ++q) {
            const half_t h = (half_t)((float)q * (float)most);                                  // exact in 32 bits, rounded once
            const double left = (double)q * (double)(float)d - (double)(float)h;                // exact in 64
            snprintf(what, sizeof what, "%d times scale %x\n", q, bits);
            if (!(fabs((double)(float)h) <= 65504.) || (double)(float)(half_t)left != left) wrong("not held: ");
        }
    }
    return 0;
}
""")
