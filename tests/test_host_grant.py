"""CPU test of csrc/grant.cuh: host threads that raise one kernel's shared-memory limit
to different sizes leave the limit at the largest that was granted."""
from __future__ import annotations

import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "momij_b200", "csrc")

SOURCE = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include "grant.cuh"

int main() {
    int granted = 0, refused = 0;
    std::atomic<int> limit{0}, started{0};
    // The larger setting is slow to be recorded; the smaller one comes in between.
    auto set = [&](int size) {
        limit = size;
        ++started;
        if (size == 100) std::this_thread::sleep_for(std::chrono::milliseconds(200));
        return true;
    };
    std::thread large([&] { momij::grant_at_least(granted, 100, set); });
    while (!started) std::this_thread::yield();
    std::thread small([&] { momij::grant_at_least(granted, 60, set); });
    large.join();
    small.join();
    if (limit < granted || granted != 100) return std::printf("limit %d, granted %d\n", limit.load(), granted), 1;
    if (!momij::grant_at_least(granted, 80, [&](int) { return ++refused, false; }) || refused) return std::printf("asked again\n"), 1;
    if (momij::grant_at_least(granted, 120, [&](int) { return false; }) || granted != 100) return std::printf("recorded a refusal\n"), 1;
    return 0;
}
"""


def test_limits_from_several_threads(tmp_path):
    src, exe = tmp_path / "grant.cpp", tmp_path / "grant"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
