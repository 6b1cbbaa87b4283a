"""What the residual's norm asks of a workgroup: its launches, compiled against a stand-in for the runtime, with the LDS that a launch asks for and that the kernel has of itself within what
the kernel may take (64 KB, unless more was asked for).  No GPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "machx_inference_engine_amd", "csrc")

PROGRAM = r"""
#include "mxq_host.h"
#include <map>
#include <stdio.h>
#include <stdlib.h>
#include "../../include/mxq.h"
namespace mxq { thread_local int g_last_hip_error = 0; }
static std::map<const void*, int> allowed;
extern "C" hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
extern "C" hipError_t hipGetLastError() { return hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute, int n) { allowed[f] = n; return hipSuccess; }
static uint32_t launched, threads, asked, most;
template <class K> static void record(K kernel, dim3 block, uint32_t lds) {
    ++launched;
    threads = block.x;
    asked = lds;
    const void* f = reinterpret_cast<const void*>(kernel);
    most = allowed.count(f) ? allowed[f] : 65536 - STATIC;
}
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) record(kernel, block, lds)
namespace mxq {
typedef _Float16 half_t;
CONSTANTS
template <bool HALVES, bool FAR> void add_norm_kernel(SumArgs) { static int n; n += HALVES + 2 * FAR; }
template <int LANES, bool HALVES> void add_norm_short_kernel(SumArgs) { static int n; n += LANES + HALVES; }
template <bool B> struct Bool { static constexpr bool value = B; };
}
using namespace mxq;
extern "C" {
LAUNCH
}
int main() {
    uint16_t* p = reinterpret_cast<uint16_t*>(4096);
    for (int halves = 0; halves < 2; ++halves)
        for (uint32_t hidden = 32; hidden <= 70000; hidden += 32) {
            launched = 0;
            const int rc = mx_add_rms_norm_f32w_q8(nullptr, p, p, reinterpret_cast<float*>(p), p, p, p, 3, hidden, 1e-5f, halves);
            if (rc || launched != 1 || threads > 1024 || asked > most || asked + STATIC > 160 * 1024) {
                printf("hidden %u: status %d, %u threads, %u + %d bytes of LDS, %u allowed\n", hidden, rc, threads, asked, STATIC, most);
                return 1;
            }
        }
    return 0;
}
"""


def part(text, begin, end):
    assert text.count(begin) == 1, begin
    i = text.index(begin)
    return text[i:text.index(end, i)]


def test_lds(tmp_path):
    text = open(os.path.join(CSRC, "producers.hip")).read()
    kernel = part(text, "constexpr uint32_t kSumThreads", "\n}\n")
    assert kernel.count("__shared__ float red[kSumThreads / 32]") == 1 and kernel.count("__shared__") == 2      # the other one is what a launch asks for
    program = PROGRAM.replace("CONSTANTS", part(text, "struct SumArgs {", "\n};\n") + "\n};\n" + kernel[:kernel.index("template")]).replace(
        "LAUNCH", part(text, "int mx_add_rms_norm_f32w_q8(", "\n}\n") + "\n}\n")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(program)
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "c++", "-D__HIP_PLATFORM_AMD__", "-DSTATIC=16", "-std=c++17", "-I", CSRC, "-I", "/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
