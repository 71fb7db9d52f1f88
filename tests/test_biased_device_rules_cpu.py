"""Device functions of the attention with changed scores that only search and count, compiled for the host from their sources.  The 32 lanes of a
warp are 32 contexts that take turns at every collective; every load is checked against the array it is for."""
import ctypes
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "flash-sparse-attention_b200", "csrc")

HARNESS = r"""
#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstring>
#include <functional>
#include <ucontext.h>
using std::max; using std::min;
#define __device__
#define __forceinline__ inline
#define __restrict__ __restrict

// ---- a warp
static ucontext_t home, ctx[32];
static char stacks[32][1 << 16];
static int me, slots[2][32], steps[32];
static bool over[32];
static std::function<void(int)> body;
static void enter() { const int lane = me; body(lane); over[lane] = true; swapcontext(&ctx[lane], &home); }
static const int* together(int v) {
    const int lane = me, at = steps[lane]++ & 1;
    slots[at][lane] = v;
    swapcontext(&ctx[lane], &home);
    return slots[at];
}
static bool warp(std::function<void(int)> f) {      // false: the lanes do not meet as often as one another
    body = std::move(f);
    for (int i = 0; i < 32; ++i) {
        steps[i] = 0; over[i] = false;
        getcontext(&ctx[i]);
        ctx[i].uc_stack.ss_sp = stacks[i]; ctx[i].uc_stack.ss_size = sizeof stacks[i]; ctx[i].uc_link = nullptr;
        makecontext(&ctx[i], enter, 0);
    }
    for (bool any = true; any;) {
        any = false;
        for (me = 0; me < 32; ++me)
            if (!over[me]) { any = true; swapcontext(&home, &ctx[me]); }
        for (int i = 1; i < 32; ++i)
            if (over[i] != over[0] || steps[i] != steps[0]) return false;
    }
    return true;
}
static unsigned __ballot_sync(unsigned, bool v) { const int* s = together(v); unsigned m = 0; for (int i = 0; i < 32; ++i) m |= (unsigned)s[i] << i; return m; }
static int __reduce_add_sync(unsigned, int v) { const int* s = together(v); int r = 0; for (int i = 0; i < 32; ++i) r += s[i]; return r; }
static int __reduce_max_sync(unsigned, int v) { const int* s = together(v); return *std::max_element(s, s + 32); }
static int __shfl_sync(unsigned, int v, int from) { const int* s = together(v); return s[from & 31]; }
static int __clz(unsigned v) { return v ? __builtin_clz(v) : 32; }
static int __ffs(unsigned v) { return __builtin_ffs((int)v); }
static int __popc(unsigned v) { return __builtin_popcount(v); }

// ---- loads of the arrays [0, n) that are open
static const int32_t* arrays[2];
static int entries, outside;
static int __ldcg(const int32_t* p) {
    for (const int32_t* a : arrays)
        if (p >= a && p < a + entries) return *p;
    ++outside;
    return 0;
}
"""


def function(name, head):
    """The text of a device function of a header, from its head on."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    at = text.index(head)
    depth, end = 0, text.index("{", at)
    while True:
        depth += (text[end] == "{") - (text[end] == "}")
        end += 1
        if depth == 0:
            return text[at:end] + ("" if "struct" not in head else ";") + "\n"


def build(tmp_path, code):
    (tmp_path / "host.cpp").write_text(HARNESS + code)
    subprocess.run(["g++", "-O1", "-g0", "-std=c++17", "-fwrapv", "-shared", "-fPIC", "-o", str(tmp_path / "host.so"), str(tmp_path / "host.cpp")], check=True)
    return ctypes.CDLL(str(tmp_path / "host.so"))


SEARCH = r"""
extern "C" int places(const int32_t* cu_q, const int32_t* cu_k, int B, int TPT, int n, int* out) {
    arrays[0] = cu_q; arrays[1] = cu_k; entries = B + 1; outside = 0;
    for (int rank = 0; rank < n; ++rank) {
        int got[32][3];
        if (!warp([&](int lane) { find_ranked_tile(cu_q, cu_k, B, TPT, rank, lane, got[lane][0], got[lane][1], got[lane][2]); })) return -1;
        for (int i = 1; i < 32; ++i)
            if (memcmp(got[i], got[0], sizeof got[0])) return -2;
        memcpy(out + 3 * rank, got[0], sizeof got[0]);
    }
    return outside;
}
"""


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    with open(os.path.join(CSRC, "sel_common.cuh")) as f:
        most = re.search(r"constexpr int kRankedSeqs = \d+;", f.read()).group(0)
    return build(tmp_path_factory.mktemp("search"), most + "\n" + function("sel_common.cuh", "__device__ __forceinline__ void find_ranked_tile(") + SEARCH)


def every_tile(search, front, lens, TPT, klens=None):
    """All places of a list: (sequence, first token, tokens) of those that hold a tile, and how many are left over behind the list."""
    klens = klens or lens
    cu, cuk = [front], [0]
    for a, b in zip(lens, klens):
        cu.append(cu[-1] + a)
        cuk.append(cuk[-1] + b)
    B = len(lens)
    n = (cu[-1] + TPT - 1) // TPT + B + 2
    array = ctypes.c_int32 * (B + 1)
    out = (ctypes.c_int * (3 * n))()
    rc = search.places(array(*cu), array(*cuk), B, TPT, n, out)
    assert rc == 0, f"{rc} loads outside of the arrays" if rc > 0 else "the lanes went different ways"
    got = [tuple(out[3 * i : 3 * i + 3]) for i in range(n)]
    tiles = sorted((s, t, ne) for s, t, ne in got if s >= 0)
    want = sorted((b, cu[b] + i, min(TPT, lens[b] - i)) for b in range(B) for i in range(0, lens[b], TPT))
    assert tiles == want
    return [t for s, t, ne in got if s < 0 and ne == 0]


@pytest.mark.parametrize("TPT", [4, 32, 128])
@pytest.mark.parametrize("front", [0, 3, 9, 70, 1000])
@pytest.mark.parametrize("lens", [[1] * 33, [2, 0, 5, 90] * 9, [0] * 40 + [300] + [0] * 30, [1, 40, 0] * 140, [1] * 1100],
                         ids=["33", "36", "71", "420", "1100"])
def test_every_tile_of_many_sequences_is_found_once(search, lens, front, TPT):
    """Rows in front of the first sequence too (sequences in front of the first group that shares rows)."""
    left = every_tile(search, front, lens, TPT)
    assert left == list(range(len(left)))           # (places behind the list count on)


@pytest.mark.parametrize("TPT", [4, 128])
@pytest.mark.parametrize("front,lens,klens", [(0, [5], None), (70, [33, 0, 129, 1], None), (9, [1] * 32, None), (0, [40, 300, 7], [500, 300, 2]), (1000, [0, 0], None)])
def test_every_tile_of_few_sequences_is_found_once(search, front, lens, klens, TPT):
    left = every_tile(search, front, lens, TPT, klens)
    assert left == list(range(len(left)))


LIMITS = r"""
extern "C" void limits(int tok, int k0, int k1, int q1, int window, int prefix, int* out) {
    const Sees x = place_limits(tok, k0, k1, q1, window, prefix);
    out[0] = x.lo; out[1] = x.hi; out[2] = x.pos;
}
"""


@pytest.fixture(scope="module")
def limits(tmp_path_factory):
    text = "struct Sees { int lo, hi, pos; };\n" + function("biased.cuh", "__device__ __forceinline__ Sees place_limits(") + LIMITS
    lib = build(tmp_path_factory.mktemp("limits"), text)

    def call(*args):
        out = (ctypes.c_int * 3)()
        lib.limits(*args, out)
        return tuple(out)

    return call


LARGEST = 2 ** 31 - 1


@pytest.mark.parametrize("k0,k1,q1", [(0, 10, 10), (0, 10, 4), (5, 25, 10), (2 ** 25 - 40, 2 ** 25 - 1, 20), (3, 3, 10), (0, 4, 10)])
@pytest.mark.parametrize("window,prefix", [(-1, 0), (-1, 3), (-1, 10), (-1, LARGEST), (-1, -1), (-1, -LARGEST), (-1, -LARGEST - 1), (0, 0), (4, 0), (LARGEST, 0)])
def test_rows_that_a_token_sees(limits, k0, k1, q1, window, prefix):
    """Of its own sequence's rows, whatever stands in prefix_lens and window_size."""
    for tok in range(max(0, q1 - 8), q1):
        pos = tok + k1 - q1
        seen = [j for j in range(k0, k1) if pos >= k0 and (j <= pos or j - k0 < prefix) and (window < 0 or j >= pos - window)]
        lo, hi, at = limits(tok, k0, k1, q1, window, prefix)
        assert at == pos and list(range(lo, min(hi, lo + 10 ** 4) + 1)) == seen
        assert hi < k1


@pytest.mark.parametrize("name,kernels", [
    ("biased_attn.cu", None), ("biased_fwd.cu", None), ("biased_bwd_dq.cu", None), ("biased_bwd_dkdv.cu", None), ("biased_decode.cu", None),
    ("range_bwd_dkdv.cu", ["range_key_tiles(const", "range_plan_items(const", "range_dkdv_reduce(const"]),
])
def test_kernels_that_start_early_read_nothing_by_the_non_coherent_path(name, kernels):
    """Such a load may be moved before the wait for the kernels before, or be answered from what was there while one of them still ran.  (A breach shows only in a
    run that a load wins by chance.)"""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    for part in [text] if kernels is None else [function(name, head) for head in kernels]:
        part = re.sub(r"//[^\n]*", "", part)
        assert "__ldg(" not in part and "ld.global.nc" not in part
        assert not re.findall(r"find_seq\(|find_seq_tile\(|count_seq_tiles\(", part)       # (they load that way unless told otherwise)
