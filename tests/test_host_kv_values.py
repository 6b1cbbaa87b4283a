"""The one-token attention's kernels over fp16 values that are no numbers, run on the CPU as a GPU runs them and compared with sums in 64 bits.  No GPU."""
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
