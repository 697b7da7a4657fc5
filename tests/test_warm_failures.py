"""What the library does where a step of its start fails: the functions' own text, compiled with fakes of the CUDA calls that fail."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "suzuku-engine-q4_b200", "csrc")

FAKES = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
enum cudaError_t { cudaSuccess, cudaErrorInvalidValue };
static cudaError_t last = cudaSuccess;
static int fail_at = -1, calls = 0;
static cudaError_t step() { return calls++ == fail_at ? (last = cudaErrorInvalidValue) : cudaSuccess; }
static cudaError_t cudaGetLastError() { const cudaError_t e = last; last = cudaSuccess; return e; }
static int held = 0;
template <typename T> static cudaError_t cudaMalloc(T **p, size_t n) {
    if (step() != cudaSuccess) return last;
    *p = (T *)malloc(n);
    held++;
    return cudaSuccess;
}
static cudaError_t cudaMemset(void *p, int v, size_t n) { return step() == cudaSuccess ? (memset(p, v, n), cudaSuccess) : last; }
static cudaError_t cudaFree(void *p) { held -= p != nullptr; free(p); return cudaSuccess; }
static const char *cudaGetErrorString(cudaError_t) { return "error"; }
"""


def _function(path, head):
    """The text of a function, from its head to the brace that closes it in the head's column."""
    text = open(os.path.join(CSRC, path)).read()
    at = text.index(head)
    return text[at:text.index("\n}\n", at) + 3]


def _run(tmp_path, source):
    src, exe = str(tmp_path / "t.cpp"), str(tmp_path / "t")
    open(src, "w").write(source)
    r = subprocess.run(["g++", "-std=c++17", "-o", exe, src], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("fail_at", range(4))
def test_shared_memory_limits_of_the_4_bit_products(tmp_path, fail_at):
    """A limit that cannot be raised: the products stay on the CUDA cores, and no error is left for the next launch's check; a second
    start tries again."""
    _run(tmp_path, FAKES + r"""
namespace mmqtc { static bool warm() { return true; } }
static bool g_tc_ready = false;
template <uint32_t BN, bool PAIR> static bool tc_attr() { return step() == cudaSuccess; }
""" + _function("q4b_fp4_tc.cu", "bool tc_warm() {") + r"""
int main() {
    fail_at = %d;
    if (tc_warm() || g_tc_ready || cudaGetLastError() != cudaSuccess) return 1;
    fail_at = -1;
    return tc_warm() && g_tc_ready && cudaGetLastError() == cudaSuccess ? 0 : 2;
}
""" % fail_at)


def test_limits_are_asked_for_again_after_a_shutdown():
    text = open(os.path.join(CSRC, "q4b_fp4_tc.cu")).read()
    assert re.search(r"void q4b_fp4_shutdown\(\) \{ fp4::g_tc_ready = false; \}", text)
    assert "q4b_fp4_shutdown();" in _function("q4b_runtime.cu", 'extern "C" void q4_hip_shutdown(void) {')


@pytest.mark.parametrize("fail_at", range(4))
def test_scratch_of_the_balance_loss(tmp_path, fail_at):
    """Scratch that cannot be had: the library starts all the same, nothing is held, no error is left, and a second start tries again."""
    text = open(os.path.join(CSRC, "q4b_balance.cu")).read()
    macro = open(os.path.join(CSRC, "q4b_internal.cuh")).read()
    macro = macro[macro.index("#define Q4B_CHECK"):macro.index("while (0)\n") + 10]
    warms = ("router_tc", "mmq_tc", "fp4", "fused", "window", "elem", "mmvq", "route_small")
    _run(tmp_path, FAKES + macro + r"""
namespace balance {
constexpr uint32_t MAX_E = 1024;
struct Args {};
static uint32_t *g_done = nullptr;
static float *g_part = nullptr;
static uint32_t g_clusters = 0;
template <int NV, bool VEC> static bool launch(const Args &, uint32_t, uint32_t *most) { return step() == cudaSuccess && (*most = 18); }
}
""" + "".join(_function("q4b_balance.cu", h) for h in sorted(("bool q4b_balance_warm() {", "void q4b_balance_shutdown() {"), key=text.index))
         + "".join("static bool q4b_%s_warm() { return true; }\n" % w for w in warms) + r"""
constexpr uint32_t Q4B_XQ_SLICES = 1, Q4B_XQ_MAXLEN = 64, Q4B_MAX_TOK = 1;
struct Q4bState { int8_t *xq; float *xd; int32_t *xbs; float *xn, *logits; int32_t *r_ids; float *r_wts; int32_t *r_cnt; float *hbuf; };
static Q4bState g_q4b = {};
""" + _function("q4b_runtime.cu", "bool alloc_scratch() {") + r"""
int main() {
    fail_at = 9 + %d;                    // behind the nine buffers of the other calls
    if (!alloc_scratch()) return 1;
    if (calls <= fail_at) return 2;
    if (balance::g_done || balance::g_part || held != 9 || cudaGetLastError() != cudaSuccess) return 3;
    fail_at = -1;
    return q4b_balance_warm() && balance::g_done && balance::g_part && balance::g_clusters == 18 ? 0 : 4;
}
""" % fail_at)
