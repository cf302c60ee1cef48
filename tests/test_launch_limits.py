"""What the C ABI's calls of the largest sizes launch, without a GPU: the library's launches are taken by a recorder that is loaded ahead of the runtime, in a process of its own.

A launch has fewer than 2^32 threads in each dimension, and 65535 workgroups at most beyond the first."""
import json
import os
import subprocess
import sys

import pytest
import torch

from htr_amd import _native, build, ops

RECORDER = r"""
#include <cstddef>
struct dim3 { unsigned x, y, z; };
static unsigned seen[1 << 16][6];
static int count = 0;
extern "C" {
int hipLaunchKernel(const void*, dim3 g, dim3 b, void**, size_t, void*) {
  if (count < (1 << 16)) { unsigned* s = seen[count++]; s[0] = g.x; s[1] = g.y; s[2] = g.z; s[3] = b.x; s[4] = b.y; s[5] = b.z; }
  return 0;
}
int hipGetDevice(int* dev) { *dev = 0; return 0; }
int hipFuncSetAttribute(const void*, int, int) { return 0; }
int recorded() { return count; }
const unsigned* record() { return seen[0]; }
void forget() { count = 0; }
}
"""
# addresses are never read: nothing is launched
CALLER = r"""
import ctypes, json, sys
recorder, library, calls = sys.argv[1], sys.argv[2], json.load(sys.stdin)
r = ctypes.CDLL(recorder, mode=ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(library)
r.record.restype = ctypes.POINTER(ctypes.c_uint)
L.htr_moe_stacked_scratch_bytes.restype = ctypes.c_size_t
I, Q, P, D = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_double
p, out = P(1 << 40), []
for name, a in calls:
    r.forget()
    if name == "moe":
        tokens, top, experts, hidden, inter, kind = a
        need = L.htr_moe_stacked_scratch_bytes(Q(tokens), I(top), I(experts), I(hidden), I(inter), I(kind))
        s = p if kind >= 3 else None
        rc = -1 if need == 0 else L.htr_moe_stacked(p, I(kind if kind < 3 else 0), p, I(1), p, Q(tokens), I(top), p, s, p, s, I(experts), I(hidden), I(inter), I(kind), p, p,
                                                    ctypes.c_size_t(need), None)
    elif name == "quantize":
        rows, n, kind = a
        rc = (L.htr_quantize_int8 if kind == 4 else L.htr_quantize_e4m3)(p, Q(n), Q(rows), I(n), I(0), p, p, None)
    elif name == "norm":
        rows, n, kind = a
        rc = (L.htr_rms_norm_int8 if kind == 4 else L.htr_rms_norm)(p, Q(n), p, Q(n), p, Q(rows), I(n), D(1e-6), I(0), p, p if kind >= 3 else None, p, None)
    elif name == "route":
        tokens, experts, top, groups = a
        rc = L.htr_route(p, Q(experts), I(2), Q(tokens), I(experts), I(top), I(1), p, I(groups), I(1), I(2), I(1), D(1.0), p, p, None)
    else:
        rows, m, n, experts, kind = a
        s = p if kind >= 3 else None
        rc = L.htr_product(p, I(kind), s, p, s, None, p if experts else None, p, Q(rows), I(m), I(n), I(max(experts, 1)), I(kind), I(0), None)
    k = r.recorded()
    out.append((rc, [list(r.record()[6 * i:6 * i + 6]) for i in range(k)]))
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    folder = tmp_path_factory.mktemp("recorder")
    source, recorder = folder / "recorder.cpp", folder / "recorder.so"
    source.write_text(RECORDER)
    subprocess.check_call([os.environ.get("CXX", "g++"), "-shared", "-fPIC", "-O1", str(source), "-o", str(recorder)])

    def run(*calls):
        done = subprocess.run([sys.executable, "-c", CALLER, str(recorder), build.LIB], input=json.dumps(calls), capture_output=True, text=True, timeout=120)
        assert done.returncode == 0, done.stderr
        return json.loads(done.stdout)
    return run


def held(call, rc, seen):
    assert rc == 0 and seen, (call, rc, len(seen))
    for g in seen:
        assert all(0 < g[k] * g[3 + k] < 1 << 32 for k in range(3)) and g[1] <= 65535 and g[2] <= 65535 and g[3] * g[4] * g[5] <= 1024, (call, g)


I8, E4M3, BF16 = 4, 3, 0
LAYERS = [(1, 1, 1, 128, 128), (4096, 6, 64, 2048, 1408), (1 << 20, 64, 8, 16, 16), (1 << 21, 8, 64, 512, 2048), ((1 << 24) - 1, 3, 8, 128, 128), ((1 << 23) - 1, 64, 64, 512, 512),
          ((1 << 23) - 1, 64, 64, 512, 2048), (1 << 18, 4096, 1, 512, 512)]


@pytest.mark.parametrize("kind", [I8, E4M3, BF16])
def test_layers_of_any_size_are_launched(launches, kind):
    """Up to 2^30 pairs of tokens and experts."""
    calls = [("moe", s + (kind,)) for s in LAYERS if _native.lib().htr_moe_stacked_scratch_bytes(*s, kind) > 0]
    assert len(calls) >= (len(LAYERS) if kind == I8 else 5)
    for call, (rc, seen) in zip(calls, launches(*calls)):
        held(call, rc, seen)


def test_the_other_calls_of_any_size_are_launched(launches):
    most = (1 << 31) - 1
    calls = [(name, (rows, n, kind)) for name in ("quantize", "norm") for kind in (I8, E4M3) for rows, n in ((most, 128), (most, 8192), (3 << 21, 40960), (1, 1 << 30))]
    calls += [("norm", (most, 8192, BF16)), ("route", (most, 256, 8, 8)), ("route", (most, 1024, 16, 1)), ("route", (5, 8, 1, 1))]
    calls += [("product", a) for a in ((most - (1 << 20), 64, 512, 0, I8), (most - (1 << 20), 64, 512, 7, I8), (1, 1 << 26, 16, 0, I8), (9, 1 << 26, 128, 3, I8), (65535, 1 << 12, 512, 65535, I8))]
    for call, (rc, seen) in zip(calls, launches(*calls)):
        held(call, rc, seen)


def test_the_recorder_takes_the_launches(launches):
    """One launch to a rounding of few rows, several to one of more rows than a launch takes; none to a call that is refused."""
    few, many, refused = launches(("quantize", (5, 128, I8)), ("quantize", ((1 << 22) + 1, 128, I8)), ("quantize", (5, 24, I8)))
    assert few == [0, [[5, 1, 1, 64, 1, 1]]] and many[0] == 0 and sum(g[0] for g in many[1]) == (1 << 22) + 1 and refused == [_native.lib().htr_quantize_int8(None, 24, 5, 24, 0, None, None, None), []]


@pytest.mark.gpu
def test_a_layer_of_more_rows_than_a_launch_takes():
    """2^26 pairs of 16 hidden columns, whose rounding was 2^32 threads; experts out of range among them, whose rows are left out of it."""
    from test_int8 import assert_within, experts, moe64, randn
    gen = torch.Generator(device="cuda").manual_seed(20261209)
    T, top, E, n = 1 << 20, 64, 8, 16
    x, wt = randn(gen, T, n, dtype=torch.bfloat16), torch.rand(T, top, device="cuda", generator=gen)
    ids = torch.randint(0, E, (T, top), dtype=torch.int32, device="cuda", generator=gen)
    ids[1, 3], ids[T - 2, 60] = -1, E
    gate_up, down = experts(gen, E, n, n)
    y = ops.moe_experts_stacked(x, ids, wt, gate_up, down)
    some = torch.tensor([0, 1, 77_777, T // 2, T - 2, T - 1], device="cuda")
    assert_within(y[some], *moe64(x[some], ids[some], wt[some], gate_up, down, torch.bfloat16))
    assert y[1].isnan().all() and y[T - 2].isnan().all()
    y[1], y[T - 2] = 0, 0
    assert y.isfinite().all()
