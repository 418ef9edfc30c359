"""The prompt attention's staging of 16-bit tiles (csrc/mq_attn_prompt.hip), its own lines compiled for the host: what its
threads look through for infinities is what they loaded or cleared, whatever LDS held before, and every value of a head arrives once."""
import os
import shutil
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfy-quant-bench_amd", "csrc", "mq_attn_prompt.hip")
CXX = shutil.which("g++") or shutil.which("c++")

HEAD = r"""
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>
#define __device__
#define __forceinline__ inline
#define __builtin_amdgcn_readfirstlane(x) (x)
struct uint4 { uint32_t x, y, z, w; };
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return uint4{x, y, z, w}; }
constexpr int kDtF16 = 1, kTile = 64;
char* g_lds;
int g_lane;
uint32_t lds_offset(const void* p) { return static_cast<uint32_t>(static_cast<const char*>(p) - g_lds); }
void load_lds16(const char* src, uint32_t dst) { std::memcpy(g_lds + dst + 16 * g_lane, src, 16); }
"""

RUN = r"""
template <int DP>
struct Lds {
    alignas(16) uint16_t k[2][kTile * DP];
    uint16_t v[2][DP * kTile];
    int64_t at[3][kTile];
    int wild;
};

template <int DP, int DT>
int run(int D) {
    constexpr int KC = DP / 32, kPerKey = DP / 8;
    static Lds<DP> sm;
    struct { int D; } a{D};
    g_lds = reinterpret_cast<char*>(&sm);
    // a cache of 64 rows of D values, key 64 - x in row x; LDS full of infinities
    std::vector<uint16_t> cache(kTile * D);
    for (int x = 0; x < kTile; ++x)
        for (int d = 0; d < D; ++d) cache[x * D + d] = static_cast<uint16_t>(1 + (x * D + d) % 20000);
    const char *kbase = reinterpret_cast<const char*>(cache.data()), *vbase = kbase;
    const uint16_t inf = DT == kDtF16 ? 0x7c00 : 0x7f80;
    for (auto& half : sm.v) for (auto& x : half) x = inf;
    for (int x = 0; x < kTile; ++x) sm.at[0][x] = 2 * D * (kTile - 1 - x);
    sm.wild = 0;
    std::vector<uint16_t> got[2];
    for (int tid = 0; tid < 256; ++tid) {
@CLEAR@
    }
    for (int tid = 0; tid < 256; ++tid) {
        const int lane = tid & 63, wave = tid >> 6;
        g_lane = lane;
@STAGE@
        fetch(0, 1);
        tame_own(1);
        if (tid < 255) continue;
        // where the products look for key x, values 8 c .. of it
        for (int x = 0; x < kTile; ++x)
            for (int d = 0; d < D; ++d) {
                const uint16_t want = cache[(kTile - 1 - x) * D + d];
                if (sm.k[1][x * DP + 8 * ((d / 8) ^ kswap(x)) + d % 8] != want) return 1;
                if (sm.v[1][x * DP + 8 * ((d / 8) ^ vswap(x)) + d % 8] != want) return 2;
            }
    }
    return sm.wild ? 3 : 0;
}

int main() {
    for (int D = 8; D <= 256; D += 8) {
        const int r = D <= 64 ? run<64, 0>(D) | run<64, 1>(D) : D <= 128 ? run<128, 0>(D) | run<128, 1>(D) : run<256, 0>(D) | run<256, 1>(D);
        if (r) {
            std::printf("D %d: %s\n", D, r == 3 ? "values that no load wrote are looked through" : "a value is not in its place");
            return 1;
        }
    }
    std::puts("all");
    return 0;
}
"""


def between(text, first, last):
    i = text.index(first)
    return text[i: text.index(last, i)]


@pytest.mark.skipif(CXX is None, reason="no C++ compiler")
def test_staged_values(tmp_path):
    with open(SRC) as f:
        text = f.read()
    wild = between(text, "template <int DT>\n__device__ __forceinline__ bool has_wild", "// 0: +infinity")
    stage = between(text, "    const int slot = tid % kPerKey;", "    // int8 caches: the tile whose codes")
    clear = between(text, "            if (8 * kPerKey > a.D)", "        }\n        __syncthreads();")
    src, exe = tmp_path / "tiles.cpp", tmp_path / "tiles"
    src.write_text(HEAD + wild + RUN.replace("@STAGE@", stage).replace("@CLEAR@", clear))
    subprocess.run([CXX, "-std=c++17", "-O1", "-w", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "all", out.stdout
