"""The workspace of the calls without a store (joule_amd/csrc/jm_plugin_ws.h),
compiled on the host with g++: a call holds its stream's buffer until all its
kernels are enqueued, so that two host threads on one stream cannot put the
kernels of one call between those of another; threads on other streams and
devices do not wait for it."""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "joule_amd" / "csrc"

DRIVER = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include "jm_plugin_ws.h"

static int fails = 0;
#define CHECK(c) do { if (!(c)) { std::printf("FAIL line %d: %s\n", __LINE__, #c); fails++; } } while (0)

// what the entry points do: take the buffer, enqueue three kernels one by one
static void call(jm::PluginBufs& bufs, void* st, int who, std::vector<int>& stream) {
    jm::PluginWs ws;
    jm::PluginBuf& b = bufs.of(0, st);
    ws.held = std::unique_lock<std::mutex>(b.mu);
    for (int k = 0; k < 3; k++) {
        stream.push_back(who);
        std::this_thread::sleep_for(std::chrono::microseconds(20));
    }
}

int main() {
    jm::PluginBufs bufs;
    int s0, s1;
    CHECK(&bufs.of(0, &s0) == &bufs.of(0, &s0));
    CHECK(&bufs.of(0, &s0) != &bufs.of(1, &s0));
    CHECK(&bufs.of(0, &s0) != &bufs.of(0, &s1));
    CHECK(&bufs.of(0, nullptr) == &bufs.of(0, nullptr));

    std::vector<int> stream;
    std::vector<std::thread> t;
    for (int who = 0; who < 4; who++)
        t.emplace_back([&, who] { for (int i = 0; i < 100; i++) call(bufs, &s0, who, stream); });
    for (auto& x : t) x.join();
    CHECK(stream.size() == 1200);
    for (size_t i = 0; i + 2 < stream.size(); i += 3) CHECK(stream[i] == stream[i + 1] && stream[i] == stream[i + 2]);

    // held by this thread: another stream's and another device's are free, this one's is not
    {
        jm::PluginWs ws;
        ws.held = std::unique_lock<std::mutex>(bufs.of(0, &s0).mu);
        std::thread([&] {
            CHECK(!bufs.of(0, &s0).mu.try_lock());
            CHECK(bufs.of(0, &s1).mu.try_lock());
            bufs.of(0, &s1).mu.unlock();
            CHECK(bufs.of(1, &s0).mu.try_lock());
            bufs.of(1, &s0).mu.unlock();
        }).join();
    }
    std::thread([&] { CHECK(bufs.of(0, &s0).mu.try_lock()); bufs.of(0, &s0).mu.unlock(); }).join();
    std::printf("%d failures\n", fails);
    return fails != 0;
}
"""


def test_a_call_holds_its_streams_buffer(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    src = tmp_path / "ws_lock.cpp"
    src.write_text(DRIVER)
    exe = tmp_path / "ws_lock"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-pthread", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_every_caller_keeps_it_over_its_launches():
    """Each entry point that takes the workspace has it in a variable of its
    own scope, not in a block that ends before its launches."""
    n = 0
    for f in sorted(CSRC.glob("*.hip")):
        text = f.read_text()
        at = text.find("jm::PluginWs ws;")
        while at >= 0:
            end = text.find("\n}\n", at)
            body = text[at:end]
            line = text[text.rfind("\n", 0, at) + 1:at]
            assert line == "    ", f"{f.name}: the workspace is not at the function's own level"
            assert "plugin_ws(" in body and "launch_" in body
            n += 1
            at = text.find("jm::PluginWs ws;", at + 1)
    assert n == 4
