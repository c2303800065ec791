"""CPU check of the sums that the waves of a row exchange through LDS in the layer norm's kernels (`row_sum`, csrc/mm_layer_norm.hip).

The function is compiled for the host out of its source, a thread for each wave and a barrier in the place of __syncthreads that
holds one wave back behind every barrier until all others wait at the next one (or are done). Then that wave reads as late as it
may: a sum whose place is written for the next one too comes out wrong, every time. The kernels' sequences are run, one value or two
at a time, in LDS of the size that they declare, with words behind it that have to stay."""
import pathlib
import re
import subprocess

import pytest

SOURCE = pathlib.Path(__file__).resolve().parents[1] / "motif-mamba_amd" / "csrc" / "mm_layer_norm.hip"

HOST = r"""
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>
#include <vector>
#define __device__
#define __forceinline__ inline
struct { unsigned x; } thread_local threadIdx;
static std::mutex m;
static std::condition_variable cv;
static int waves, late, here, done, turn;

template <int N> float group_sum(float x) { return x; }   // a wave's lanes: the first one has the wave's sum
static float __shfl_xor(float, int) { return 0.f; }
static void __syncthreads() {
    std::unique_lock<std::mutex> l(m);
    const int mine = turn;
    if (++here == waves) {
        here = 0;
        ++turn;
    }
    cv.notify_all();
    cv.wait(l, [&] { return turn != mine; });
    if (int(threadIdx.x / 64) == late) cv.wait(l, [&] { return here + done == waves - 1; });
}

%(row_sum)s

template <int W, int N> static int one(int n, int wave, float *buf, int &half) {
    float x[N], want[N] = {};
    for (int i = 0; i < N; ++i) {
        x[i] = float(1 + wave + 10 * i + 100 * n);
        for (int w = 0; w < W; ++w) want[i] += float(1 + w + 10 * i + 100 * n);
    }
    row_sum<W>(x, buf, half);
    int bad = 0;
    for (int i = 0; i < N; ++i) bad += x[i] != want[i];
    return bad;
}
template <int W> static int run(int size, const char *sums, int rows) {
    std::vector<float> buf(size + 64, -1.f);
    std::vector<int> bad(W, 0);
    std::vector<std::thread> all;
    waves = W;
    here = done = turn = 0;
    for (int w = 0; w < W; ++w)
        all.emplace_back([&, w] {
            threadIdx.x = 64 * w;
            int half = 0, n = 0;
            for (int r = 0; r < rows; ++r)
                for (const char *s = sums; *s; ++s, ++n) bad[w] += *s == '1' ? one<W, 1>(n, w, buf.data(), half) : one<W, 2>(n, w, buf.data(), half);
            std::lock_guard<std::mutex> l(m);
            ++done;
            cv.notify_all();
        });
    int res = 0;
    for (auto &t : all) t.join();
    for (int b : bad) res += b;
    for (int i = 0; i < 64; ++i) res += 1000 * (buf[size + i] != -1.f);
    return res;
}
int main() {
    constexpr int W = 4;
    struct { const char *name; int size; const char *sums; int rows; } cases[] = {
        {"forward", %(ln_fwd)s, "11", 1}, {"forward, rms", %(ln_fwd)s, "1", 1},
        {"backward", %(ln_bwd)s, "112", 5}, {"backward, rms", %(ln_bwd)s, "12", 5}};
    for (auto &c : cases)
        for (late = -1; late < W; ++late) std::printf("%%s; %%d; %%d\n", c.name, late, run<W>(c.size, c.sums, c.rows));
}
"""


@pytest.fixture(scope="module")
def wrong(tmp_path_factory):
    """{(kernel, the wave that is late or -1): values that came out wrong}"""
    text = SOURCE.read_text()
    parts = {"row_sum": re.search(r"^template <int W, int N>\n__device__ __forceinline__ void row_sum\(.*?^}", text, re.M | re.S).group(0)}
    for kernel in ("ln_fwd", "ln_bwd"):
        parts[kernel] = re.search(rf"^__global__ void [^\n]* {kernel}\(.*?__shared__ float buf\[(.*?)\][,;]", text, re.M | re.S).group(1)
    d = tmp_path_factory.mktemp("sums")
    (d / "sums.cpp").write_text(HOST % parts)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-pthread", "-Wno-unknown-pragmas", str(d / "sums.cpp"), "-o", str(d / "sums")])
    out = subprocess.run([str(d / "sums")], stdout=subprocess.PIPE, check=True, timeout=60).stdout.decode()
    return {(a, int(b)): int(n) for a, b, n in (line.split("; ") for line in out.splitlines())}


@pytest.mark.parametrize("late", [-1, 0, 1, 2, 3])
@pytest.mark.parametrize("kernel", ["forward", "forward, rms", "backward", "backward, rms"])
def test_a_late_wave_takes_its_own_sums(wrong, kernel, late):
    assert wrong[kernel, late] == 0
