"""The order of the w4a16 kernel's loads and products (csrc/mq_w4a16_runs.h), run on the host: whatever the cut into chunks
and tiles, a step's products take the weights that were loaded for it, and every step of every tile is taken once. The
loops below are the kernel's, with a load and a product replaced by a record."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfy-quant-bench_amd", "csrc")
CXX = shutil.which("g++") or shutil.which("c++")

PROGRAM = r"""
#define __host__
#define __device__
#define __forceinline__ inline
#include "mq_w4a16_runs.h"
#include <cstdio>
#include <vector>

// The error, if there is one: K values of which `chunk` are staged at a time, tiles first, first + stride, ...
template <int W, int KB, bool THROUGH>
const char* follow(int K, int chunk, int first, int tiles, int stride) {
    struct Step { int tile = -1, blk = -1; };
    const int blocks = (K + 127) / 128, chunk_steps = chunk / 128;
    const int per = mq::w4_share<W>(chunk_steps), run = mq::w4_run<KB>(per);
    std::vector<int> taken(static_cast<size_t>(tiles) * blocks, 0);
    for (int wave = 0; wave < W; ++wave) {
        Step place[KB];
        mq::W4Fetch<THROUGH> ahead(first, wave, per);
        auto fetch_next = [&](int i) {
            if (ahead.any(per, blocks, tiles)) {
                if (ahead.blk < 0 || ahead.tile < 0) return;
                place[i].tile = ahead.tile;
                place[i].blk = ahead.blk;
            }
            ahead.next(wave, per, run, chunk_steps, blocks, stride);
        };
        for (int i = 0; i < KB; ++i) fetch_next(i);
        int tile = first;
        do {
            for (int k0 = 0; k0 < K; k0 += chunk) {
                const int b0 = k0 / 128 + wave * per, chunk_end = (k0 + chunk) / 128;
                const int b1 = b0 + per < chunk_end ? b0 + per : chunk_end, b2 = b1 < blocks ? b1 : blocks;
                for (int b = b0; b < b0 + run; b += KB)
                    for (int i = 0; i < KB; ++i) {
                        if (b + i < b2) {
                            if (place[i].tile != tile || place[i].blk != b + i) return "another step's weights";
                            ++taken[static_cast<size_t>(tile) * blocks + b + i];
                        }
                        fetch_next(i);
                    }
            }
            tile += stride;
        } while (THROUGH && tile < tiles);
    }
    for (int t = first; t < tiles; t += stride) {
        for (int b = 0; b < blocks; ++b)
            if (taken[static_cast<size_t>(t) * blocks + b] != 1) return "a step that is not taken once";
        if (!THROUGH) break;
    }
    return nullptr;
}

template <int W, int KB, bool THROUGH>
long cuts(int K) {
    long n = 0;
    for (int unit : {128, 1024}) {
        const int all = (K + unit - 1) / unit * unit;
        int step = W * KB * 128;
        while (step % unit) step += W * KB * 128;
        for (int chunk = all; chunk > 0; chunk = chunk == all ? (all - 1) / step * step : chunk > 4 * step ? chunk / step / 2 * step : chunk - step)
            for (int tiles : {1, 2, 3, 7, 16}) {
                const int stride = THROUGH ? 3 : tiles;
                for (int first = 0; first < (THROUGH ? 3 : 1) && first < tiles; ++first, ++n)
                    if (const char* what = follow<W, KB, THROUGH>(K, chunk, first, tiles, stride)) {
                        std::printf("W %d KB %d K %d chunk %d first %d tiles %d: %s\n", W, KB, K, chunk, first, tiles, what);
                        return -1;
                    }
            }
    }
    return n;
}

int main() {
    long n = 0;
    for (int K = 32; K <= 32768; K += K < 9000 ? 32 : 1184) {
        const long a = cuts<8, 4, true>(K), b = cuts<8, 4, false>(K), c = cuts<4, 4, false>(K), d = cuts<4, 3, false>(K);
        if (a < 0 || b < 0 || c < 0 || d < 0) return 1;
        n += a + b + c + d;
    }
    std::printf("%ld cuts\n", n);
    return 0;
}
"""


@pytest.mark.skipif(CXX is None, reason="no C++ compiler")
def test_every_product_takes_its_own_weights(tmp_path):
    src, exe = tmp_path / "runs.cpp", tmp_path / "runs"
    src.write_text(PROGRAM)
    subprocess.run([CXX, "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout.split()[0]) > 20000
