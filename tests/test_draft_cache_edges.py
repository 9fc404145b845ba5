"""The library's own refusals of the operators of a cache that is drafted into and thinned out; no GPU needed."""
import os
import re
import shutil
import subprocess

import pytest
import torch

from lightllm_b200.csrc import build, ops

T, S, L, SLOTS, HQ, HKV, HD, PAGES, PAGE, WIDTH = 6, 2, 3, 32, 4, 2, 16, 3, 8, 4


def refusal(call, pack, *numbers):
    """What the library says to a call that it refuses before anything is launched."""
    assert call(pack(*numbers), 0) != 0
    return ops.lib().llb_last_error().decode()


NAMES = ("q", "k_cache", "v_cache", "out", "mass", "mass_in", "span_row", "span_len", "span_pos", "block_table", "scratch", "flag", "tokens", "parents",
        "targets", "path", "count", "next_token", "lengths", "ends", "positions", "positions_out")
SIZES = dict(q=T * HQ * HD * 4, out=T * HQ * HD * 4, k_cache=SLOTS * HKV * HD * 4, v_cache=SLOTS * HKV * HD * 4, mass=HKV * SLOTS * 4, mass_in=HKV * SLOTS * 4,
             span_row=S * 4, span_len=S * 4, span_pos=S * 4, block_table=S * PAGES * 4)
ARENA = torch.zeros(1 << 21, dtype=torch.uint8)


def memory():
    """An address for every range of the calls, by name, all far from each other."""
    return {name: ARENA.data_ptr() + 65536 * (i + 1) for i, name in enumerate(NAMES + ("mask",))}


def attention_call(at, mass):
    span = [at[x] for x in ("q", "k_cache", "v_cache", "out", "span_row", "span_len", "span_pos", "block_table", "scratch", "flag")]
    span += [ops.F32, S, T, PAGES, PAGE, SLOTS, HQ, HKV, HD, 0.25]
    if mass:
        return ops.lib().llb_paged_attention_mass, ops._ATTENTION_MASS, *span, at["mass_in"], at["mass"], 3, 0
    return ops.lib().llb_tree_attention, ops._TREE_ATTENTION, *span, at["mask"], 1, 0


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("under", ["q", "k_cache", "v_cache", "span_row", "span_len", "span_pos", "block_table"])
def test_attention_refuses_results_over_what_it_reads(mass, under):
    at = memory()
    for written in ["out", "mass"] if mass else ["out"]:
        for moved in (0, 4, SIZES[under] - 4, 4 - SIZES[written]):
            there = dict(at, **{written: at[under] + moved})
            assert refusal(*attention_call(there, mass)).endswith(f"{written} must not lie over {under}")


def test_trees_refuse_results_over_their_masks():
    at = memory()
    assert refusal(*attention_call(dict(at, out=at["mask"]), False)).endswith("out must not lie over mask")


def test_weights_go_on_in_the_same_plane_or_in_one_of_its_own():
    """Blocks add a key's sum to what another key's place may already have lost, if the two planes are some places apart."""
    at = memory()
    for moved in (4, -4, SIZES["mass"] - 4):
        assert refusal(*attention_call(dict(at, mass=at["mass_in"] + moved), True)).endswith("mass must not lie over mass_in")
    assert refusal(*attention_call(dict(at, mass=at["out"]), True)).endswith("out must not lie over mass")


def commit_call(at):
    order = ("tokens", "parents", "targets", "k_cache", "v_cache", "span_row", "span_len", "span_pos", "block_table", "path", "count", "next_token")
    return ops.lib().llb_tree_commit, ops._TREE_COMMIT, *(at[x] for x in order), S, T, 1, PAGES, PAGE, SLOTS, HKV * HD * 4, WIDTH


@pytest.mark.parametrize("written", ["k_cache", "v_cache", "path", "count", "next_token"])
@pytest.mark.parametrize("under", ["tokens", "parents", "targets", "span_row", "span_len", "span_pos", "block_table", "v_cache", "path"])
def test_commit_refuses_results_over_what_it_reads(written, under):
    """Every block finds the path for itself, some when others have written theirs."""
    if written == under or (written, under) == ("path", "v_cache"):
        return
    at = memory()
    said = refusal(*commit_call(dict(at, **{written: at[under]})))
    assert said.endswith(f"{written} must not lie over {under}") or said.endswith(f"{under} must not lie over {written}")


def evict_call(at, apart):
    ints = (S, 1, HKV, PAGES, PAGE, SLOTS, HD * 4, 8, 2, 4)
    order = ("k_cache", "v_cache", "mass_in", "positions", "mass", "positions_out", "lengths", "ends", "block_table")
    at = dict(at) if apart else dict(at, mass=at["mass_in"], positions_out=at["positions"])
    return ops.lib().llb_cache_evict, ops._CACHE_EVICT, *(at[x] for x in order), *ints


@pytest.mark.parametrize("written,under,moved", [
    ("mass", "mass_in", 4), ("mass", "mass_in", -4), ("positions_out", "positions", 4), ("mass", "positions", 0), ("positions_out", "mass_in", 0),
    ("mass", "positions_out", 0), ("k_cache", "v_cache", 4), ("k_cache", "mass_in", 0), ("v_cache", "positions", 0), ("k_cache", "block_table", 0),
    ("mass", "lengths", 0), ("positions_out", "ends", 0), ("mass", "k_cache", 8)])
def test_eviction_refuses_planes_that_overlap(written, under, moved):
    """Holes' weights are written while other places' are read: planes are the same or have nothing in common."""
    at = memory()
    assert "must not lie over" in refusal(*evict_call(dict(at, **{written: at[under] + moved}), True))
    if written in ("k_cache", "v_cache"):
        assert "must not lie over" in refusal(*evict_call(dict(at, **{written: at[under] + moved}), False))


@pytest.mark.parametrize("kernel", ["span_attention_tc_kernel", "span_mass_tc_kernel"])
def test_a_block_that_gives_up_waits_for_all_its_loads(kernel):
    """A load that is still on its way when its block ends writes to shared memory that the next block may own: the loader waits, with a limit, on
    every barrier that its loads complete on."""
    with open(os.path.join(build.CSRC_DIR, "span_attention_tcgen05.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[text.index(kernel + "(const __grid_constant__"):]
    body = body[:body.index("\n}\n")]
    loads = set(re.findall(r"tma_load_\dd\([^;]*?&(\w+)\[[^\]]*\]\)", body))
    waited = set(re.findall(r"(?:loads_arrive\(&|ring_arrives\()(\w+)", body))
    assert loads and waited == loads
    for bar in re.findall(r"loads_arrive\(&(\w+)\[", body):          # (named one by one: both of them)
        assert {int(i) for i in re.findall(r"loads_arrive\(&%s\[(\d)\]" % bar, body)} == set(range(int(re.search(r"%s\[(\d)\]" % bar, body).group(1))))


TWO_THREADS = r"""
#include "shared_memory.h"

#include <chrono>
#include <thread>

// A runtime whose attribute is slow to set for the smaller size: the larger one would be set meanwhile, if it could.
std::atomic<int> attribute{0}, setting{0};
extern "C" cudaError_t cudaGetDevice(int* device) { *device = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
    ++setting;
    if (bytes == 1000)
        for (int i = 0; i < 500 && attribute < 2000; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    attribute = bytes;
    return cudaSuccess;
}

int main() {
    static LlbSharedMemory room;
    static int kernel;
    bool fits[2];
    std::thread small([&] { fits[0] = room.allow(&kernel, 1000) == cudaSuccess && attribute >= 1000; });
    while (setting == 0) std::this_thread::yield();
    std::thread large([&] { fits[1] = room.allow(&kernel, 2000) == cudaSuccess && attribute >= 2000; });
    small.join();
    large.join();
    // what either launches next, and a smaller size behind them
    return fits[0] && fits[1] && attribute == 2000 && room.allow(&kernel, 1500) == cudaSuccess && attribute == 2000 ? 0 : 1;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.exists("/usr/local/cuda/include/cuda_runtime.h"), reason="g++ and the CUDA headers are needed")
def test_two_host_threads_opt_in_to_shared_memory(tmp_path):
    """Calls of different head sizes at once: the limit that one of them is about to launch with is not lowered by the other."""
    source, program = tmp_path / "threads.cpp", tmp_path / "threads"
    source.write_text(TWO_THREADS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", build.CSRC_DIR, "-I", "/usr/local/cuda/include", str(source), "-o", str(program)], check=True)
    assert subprocess.run([str(program)], timeout=60).returncode == 0


def test_kernels_of_the_drafted_cache_opt_in_that_way():
    for name in ("span_attention.cu", "span_attention_tcgen05.cu", "cache_rows.cu"):
        with open(os.path.join(build.CSRC_DIR, name)) as f:
            text = f.read()
        assert "cudaFuncSetAttribute" not in text and "LlbSharedMemory" in text, name


def test_empty_ranges_lie_over_nothing():
    """A commit's drafted tokens may be none: what their address is says nothing.  (Refused all the same here, for its path.)"""
    at = memory()
    order = ("tokens", "parents", "targets", "k_cache", "v_cache", "span_row", "span_len", "span_pos", "block_table", "path", "count", "next_token")
    there = dict(at, tokens=at["k_cache"] + 64, parents=at["path"] + 4, path=at["count"])
    said = refusal(ops.lib().llb_tree_commit, ops._TREE_COMMIT, *(there[x] for x in order), S, 0, 1, PAGES, PAGE, SLOTS, HKV * HD * 4, WIDTH)
    assert said.endswith("path must not lie over count")
