"""Taking the sequence operators' reports loses none that arrives meanwhile (host only, two threads)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The writer reports, waits until its report was taken, and reports again; the reader takes all the time.  A report that
# the reader clears without having seen it leaves the writer waiting.
PROGRAM = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include "seq_status.hpp"

int main() {
    alignas(64) static int word = 0;
    std::atomic<long> taken{0};
    std::atomic<bool> stop{false};
    std::thread reader([&] {
        while (!stop) if (ppocr::take_status(&word)) ++taken;
    });
    const auto deadline = std::chrono::steady_clock::now() + std::chrono::seconds(3);
    long reports = 0;
    bool lost = false;
    for (; reports < 2000000 && !lost; ++reports) {
        *const_cast<volatile int*>(&word) = 1;
        const auto start = std::chrono::steady_clock::now();
        while (taken.load() <= reports && !lost) lost = std::chrono::steady_clock::now() - start > std::chrono::seconds(2);
        if (std::chrono::steady_clock::now() > deadline) break;
    }
    stop = true;
    reader.join();
    std::printf("%ld reports%s\n", reports, lost ? ", one lost" : "");
    return lost;
}
"""


def test_no_report_is_lost(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs a C++ compiler")
    src = tmp_path / "take.cpp"
    src.write_text(PROGRAM)
    host = os.path.join(ROOT, "ppocr-rs_b200", "csrc", "host")
    subprocess.run(["g++", "-O2", "-std=c++17", "-pthread", "-I", host, str(src), "-o", str(tmp_path / "take")], check=True)
    run = subprocess.run([str(tmp_path / "take")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout
