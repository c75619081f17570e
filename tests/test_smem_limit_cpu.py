"""Shared-memory limits raised by several host threads at once (csrc/vxc_smem_limit.h)
over a stand-in for the CUDA runtime that takes its time, no GPU needed."""
import os
import subprocess

from _paths import ROOT

PROGRAM = r"""
#include <stdio.h>
#include <unistd.h>
#include <thread>
#include "vxc_smem_limit.h"

static std::atomic<size_t> limit_of[2];
static std::atomic<int> asked{0};
struct Fake {
    typedef int error;
    static constexpr int ok = 0;
    static int device(int *d) { return *d = 0; }
    static int limit(const void *k, size_t *n) {
        asked++;
        *n = limit_of[(size_t)k - 1];
        usleep(20000);   // another thread asks meanwhile
        return 0;
    }
    static int set_limit(const void *k, size_t n) {
        usleep(n % 2 ? 20000 : 0);   // the odd, smaller one comes last
        if (limit_of[(size_t)k - 1].exchange(n) > n) printf("limit of kernel %zu lowered to %zu\n", (size_t)k, n);
        return 0;
    }
};

int main() {
    const void *a = (const void *)1, *b = (const void *)2;
    auto allow = [](const void *k, size_t n) {
        if (vxc_smem_allow<Fake>(k, n) != 0 || (n > VXC_SMEM_DEFAULT && limit_of[(size_t)k - 1] < n))
            printf("limit %zu of kernel %zu below %zu\n", (size_t)limit_of[(size_t)k - 1], (size_t)k, n);
    };
    for (int round = 0; round < 4; round++) {
        const size_t n = 60000 + 2000 * round;
        std::thread t1(allow, a, n), t2(allow, a, n - 999), t3(allow, b, n - 999), t4(allow, b, n);
        t1.join(), t2.join(), t3.join(), t4.join();
        allow(a, n);   // and afterwards
        allow(b, n);
    }
    const int before = asked;
    allow(a, 50000);
    allow(b, 66000);
    allow(a, 48 * 1024);
    if (asked != before) printf("asked again\n");
    puts("done");
}
"""


def test_limits_are_never_lowered(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-pthread", "-I", os.path.join(ROOT, "veltrix-engine_b200", "csrc"), str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.stdout == "done\n", r.stdout
