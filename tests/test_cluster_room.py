"""What is remembered of the clusters that a device holds at once (csrc/cluster_room.h, host code without CUDA): the answers, never a failure to get them."""
from __future__ import annotations

import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-backend-but-rust_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <thread>
#include <vector>
#include "cluster_room.h"
using namespace b200q;
static ClusterRoom rooms;
static int asked = 0;
static int ask(int i, int& n, int fails) { return ++asked, n = 100 * i, i == fails ? 35 : 0; }
static void tell(int device, int fails) {
    const int* room = nullptr;
    asked = 0;
    const int rc = rooms.get(device, [&](int i, int& n) { return ask(i, n, fails); }, &room);
    printf("%d %d %d %d\n", rc, asked, room ? room[2] : -1, room ? room[8] : -1);
}
int main() {
    tell(0, 2), tell(0, 5), tell(0, 0), tell(0, 3), tell(1, 8), tell(1, 0), tell(1, 2), tell(0, 2);
    std::vector<std::thread> all;
    int wrong[8] = {};
    for (int t = 0; t < 8; ++t)
        all.emplace_back([&wrong, t] {
            for (int i = 0; i < 1000; ++i) {
                const int* room = nullptr;
                rooms.get(2 + i % 9, [&](int n, int& v) { return v = 7 * n, (i + t) % 3 == 0 ? 1 : 0; }, &room);
                if (room && (room[2] != 14 || room[8] != 56)) ++wrong[t];
            }
        });
    for (auto& t : all) t.join();
    int sum = 0;
    for (int w : wrong) sum += w;
    printf("%d\n", sum);
}
"""


def test_a_failure_is_not_remembered(tmp_path):
    src = tmp_path / "room.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-pthread", "-I" + CSRC, str(src), "-o", str(tmp_path / "room")], check=True)
    lines = subprocess.run([str(tmp_path / "room")], check=True, capture_output=True, text=True).stdout.split("\n")
    # asked until it failed; then for all seven; then no more. Devices on their own
    assert lines[:8] == ["35 1 -1 -1", "35 4 -1 -1", "0 7 200 800", "0 0 200 800", "35 7 -1 -1", "0 7 200 800", "0 0 200 800", "0 0 200 800"]
    assert lines[8] == "0"
