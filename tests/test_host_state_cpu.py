"""What can be checked on the host of the norm and projection kernels: the
launchers' state (csrc/kda_host.cuh) with a fake runtime, and the ring's
bookkeeping (csrc/kda_ring.cuh). No GPU, no kernel."""

import os
import subprocess

import pytest

from conftest import PKG_DIR

FAKE_RUNTIME = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

static thread_local int device = 0;
static std::atomic<int> attribute[128];        // by device: the last value set
static std::atomic<int> calls{0}, queries{0};
static std::atomic<bool> hold_small{false}, large_set{false};

static cudaError_t fake_get_device(int *dev) { return *dev = device, cudaSuccess; }
static cudaError_t fake_get_attribute(int *v, cudaDeviceAttr, int dev) { return ++queries, *v = 100 + dev, cudaSuccess; }
template <typename K>
cudaError_t fake_set_attribute(K, cudaFuncAttribute, int bytes) {
    ++calls;
    // A thread that asks for little stands here until the larger request has gone through, or 300 ms.
    for (int i = 0; hold_small && bytes < 1000 && !large_set && i < 300; ++i)
        std::this_thread::sleep_for(std::chrono::milliseconds(1));
    attribute[device] = bytes;
    if (bytes >= 1000) large_set = true;
    return cudaSuccess;
}
static cudaError_t pending = cudaSuccess, launch_result = cudaSuccess;   // the runtime's last error, and a launch's own
static cudaError_t fake_last_error() {
    const cudaError_t e = pending;
    pending = cudaSuccess;
    return e;
}
template <typename... P, typename... A>
cudaError_t fake_launch(const cudaLaunchConfig_t *, void (*)(P...), A &&...) {
    if (launch_result != cudaSuccess) pending = launch_result;
    return launch_result;
}
#define cudaGetLastError fake_last_error
#define cudaLaunchKernelEx fake_launch
#define cudaGetDevice fake_get_device
#define cudaDeviceGetAttribute fake_get_attribute
#define cudaFuncSetAttribute fake_set_attribute
#include "kda_host.cuh"
#undef cudaGetLastError
#undef cudaLaunchKernelEx
#undef cudaGetDevice
#undef cudaDeviceGetAttribute
#undef cudaFuncSetAttribute

static void kernel() {}
// One kernel's opt-in, as a launcher holds it.
static bool ask(int bytes) {
    static kda::OptIn opted;
    return kda::opt_in(&kernel, opted, bytes);
}
"""


def run(tmp_path, body, prelude=FAKE_RUNTIME):
    """The integers that a main() of `body` prints."""
    src, exe = tmp_path / "host.cpp", tmp_path / "host"
    src.write_text(prelude + "int main() {\n" + body + "\n}\n")
    include = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f"-I{include}", f"-I{PKG_DIR / 'csrc'}", str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout
    return [int(v) for v in out.split()]


def test_two_first_calls_leave_the_larger_opt_in(tmp_path):
    """Two host threads whose first calls of one kernel need different sizes:
    whichever is second, the kernel keeps the larger one."""
    after, again, calls = run(tmp_path, r"""
        hold_small = true;
        std::thread small([] { ask(100); });
        std::this_thread::sleep_for(std::chrono::milliseconds(50));   // inside its request by now
        std::thread large([] { ask(2000); });
        small.join(), large.join();
        const int after = attribute[0];
        const int before = calls;
        ask(2000), ask(100), ask(1500);
        printf("%d %d %d\n", after, attribute[0].load(), calls - before);
    """)
    assert after == 2000 and again == 2000 and calls == 0


def test_devices_beyond_the_table(tmp_path):
    """Device 70 takes neither device 0's opt-in nor its SM count, and keeps its own."""
    got = run(tmp_path, r"""
        const int sms = kda::sm_count();
        ask(2000);
        device = 70;
        const int far = kda::sm_count();
        ask(2000);
        ask(100);
        const int opted = attribute[70];
        device = 0;
        printf("%d %d %d %d %d\n", sms, far, opted, calls.load(), kda::sm_count());
    """)
    assert got == [100, 170, 2000, 2, 100]


def test_a_launch_answers_for_itself(tmp_path):
    """An error that another call left behind is neither this launch's nor taken from whom it is for; a launch that
    fails reports its own and leaves none behind."""
    got = run(tmp_path, r"""
        const auto launch = [] { return kda::launch_overlapped(&kernel, dim3(1), 32, 0, 1, nullptr); };
        pending = cudaErrorHostMemoryAlreadyRegistered;
        const int fine = launch(), left = pending;
        pending = cudaSuccess, launch_result = cudaErrorInvalidValue;
        const int failed = launch();
        printf("%d %d %d %d\n", fine == cudaSuccess, left == cudaErrorHostMemoryAlreadyRegistered,
               failed == cudaErrorInvalidValue, pending == cudaSuccess);
    """)
    assert got == [1, 1, 1, 1]


RING = r"""
#include <cstdio>
#include <vector>
#include "kda_ring.cuh"
"""


@pytest.mark.parametrize("stages", [2, 3, 6, 16])
def test_ring_after_an_expired_wait(tmp_path, stages):
    """Turn `stuck`'s copies do not land, as warp 0 of the norms' ring kernels goes
    through its turns: no stage is filled twice without having been met, and what
    is waited for at the end is all that is in flight, each on its own parity."""
    got = run(tmp_path, r"""
        int bad = 0, cases = 0;
        for (int total = 1; total <= 40; ++total)
            for (int stuck = 0; stuck <= total; ++stuck) {   // == total: nothing expires
                const int stages = %d;
                const kda::RingTurns turns = {stages};
                std::vector<int> held(stages, -1), uses(stages, 0);   // the turn whose copies a stage waits for
                const auto fill = [&](int turn) {
                    if (turn >= total) return;                  // past the last row: nothing asked for
                    bad += held[turn %% stages] >= 0;
                    held[turn %% stages] = turn, ++uses[turn %% stages];
                };
                for (int i = 0; i < stages; ++i) fill(i);
                int turn = 0;
                for (; turn < total && turn != stuck; ++turn) {
                    held[turn %% stages] = -1;                  // met
                    fill(turn + stages);
                }
                std::vector<bool> waited(total, false);
                for (const int end = turns.end_in_flight(turn); turn < end && turn < total; ++turn) {
                    waited[turn] = true;
                    bad += turns.stage(turn) != turn %% stages || held[turn %% stages] != turn;
                    bad += static_cast<int>(turns.parity(turn)) != ((uses[turn %% stages] - 1) & 1);
                }
                for (int s = 0; s < stages; ++s) bad += held[s] >= 0 && !waited[held[s]];
                ++cases;
            }
        printf("%%d %%d\n", bad, cases);
    """ % stages, RING)
    assert got == [0, 860]


def test_schemas_say_which_results_may_be_none():
    """scale without an e4m3 output, the sum without a residual."""
    import torch
    import sgl_glm53_ascend_ops  # noqa: F401

    ns = torch.ops.sgl_glm53_ascend
    assert str(ns.kda_rmsnorm.default._schema).endswith("bool fp8=False) -> (Tensor, Tensor?, Tensor?)")
    assert str(ns.kda_gated_rmsnorm.default._schema).endswith("bool fp8=False) -> (Tensor, Tensor?)")


def test_overlapped_kernels_take_no_read_only_loads():
    """Kernels that start while the one before them runs (launch_overlapped) may read what that one still writes. The
    read-only path needs memory that nobody writes for as long as the kernel runs, so their sources do not use it."""
    sources = sorted((PKG_DIR / "csrc").glob("*.cu"))
    overlapped = [p for p in sources if "launch_overlapped(" in p.read_text()]
    assert {p.name for p in overlapped} == {"kda_norm.cu", "kda_linear.cu"}
    for path in overlapped + [PKG_DIR / "csrc" / "kda_rows.cuh", PKG_DIR / "csrc" / "kda_ring.cuh"]:
        text = path.read_text()
        for word in ("__ldg(", "ld.global.nc", "__restrict__", "load_bf16x4(", "load_f32x4("):
            assert word not in text, f"{path.name}: {word}"
