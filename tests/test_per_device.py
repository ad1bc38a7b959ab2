"""Shared memory is reserved once on every device, not once a process: the helper compiled for the host, and the launches of the 4-bit cache's
attention that have to use it (no GPU)."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qwen_inference_lab_b200" / "csrc"
PROGRAM = r"""
#include "per_device.cuh"
#include <cstdio>
#include <initializer_list>
#include <thread>
int main() {
    static QilPerDevice ready;
    int calls = 0, answer = 0;
    auto set = [&] { ++calls; return answer; };
    for (int device : {0, 1, 0, 1, 63, 63}) printf("%d ", (ready.once(device, set), calls));       // 1 2 2 2 3 3
    answer = 7;
    printf("%d ", ready.once(2, set));                            // fails: 7
    answer = 0;
    printf("%d ", ready.once(2, set));                            // tried again: 0
    printf("%d ", calls);                                           // 5
    ready.once(2, set);
    printf("%d ", calls);                                           // 5
    for (int device : {-1, 64, 64}) ready.once(device, set);        // unknown devices: every time
    printf("%d ", calls);                                           // 8
    static QilPerDevice shared[1];
    std::thread threads[8];
    std::atomic<int> wrong{0};
    for (int i = 0; i < 8; ++i) threads[i] = std::thread([&, i] {
        bool mine = false;                                          // whoever goes on has seen its own device set up
        for (int turn = 0; turn < 1000; ++turn) wrong += shared[0].once(i % 4, [&] { mine = true; return 0; }) != 0;
        wrong += !mine && !shared[0].done[i % 4];
    });
    for (auto& thread : threads) thread.join();
    printf("%d\n", wrong.load());
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_once_on_every_device(tmp_path):
    (tmp_path / "once.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-pthread", f"-I{CSRC}", str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once")], check=True)
    out = subprocess.run([str(tmp_path / "once")], capture_output=True, text=True, check=True, timeout=60).stdout
    assert out.split() == "1 2 2 2 3 3 7 0 5 5 8 0".split()


@pytest.mark.parametrize("name", ["attention_tc.cu", "kv4_attention.cu", "kv4_attention_mma.cu"])
def test_no_launch_reserves_once_a_process(name):
    """Every reservation of these files stands inside a ``once`` of the current device."""
    source = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.search(r"static\s+bool", source)
    reserved = [m.start() for m in re.finditer(r"cudaFuncSetAttribute\(", source)]
    begun = [source.rfind(".once(qil_device(), [", 0, at) for at in reserved]
    assert reserved and all(start >= 0 and source.count(";", start, at) <= 1 for start, at in zip(begun, reserved))
