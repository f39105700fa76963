"""Several host threads on one stream: a call that hands results from one launch
to the next through the stream's workspace keeps its launches together.

On the CPU, in a process whose HIP runtime is a stand-in: its launches note which
thread made them, wait a little and run nothing, its memory is the host's."""
import os
import subprocess
import sys

import pytest

from eredu_amd.build import LIB_PATH

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = r"""
#include <pthread.h>
#include <stdlib.h>
#include <time.h>
static pthread_mutex_t mu = PTHREAD_MUTEX_INITIALIZER;
static unsigned long who[4096];
static int count;
typedef struct { unsigned x, y, z; } dim;
static __thread struct { dim g, b; size_t lds; void* stream; } config;
int __hipPushCallConfiguration(dim g, dim b, size_t lds, void* stream) {
    config.g = g, config.b = b, config.lds = lds, config.stream = stream;
    return 0;
}
int __hipPopCallConfiguration(dim* g, dim* b, size_t* lds, void** stream) {
    *g = config.g, *b = config.b, *lds = config.lds, *stream = config.stream;
    return 0;
}
int hipLaunchKernel(const void* f, dim g, dim b, void** args, size_t lds, void* stream) {
    pthread_mutex_lock(&mu);
    if (count < 4096) who[count++] = (unsigned long)pthread_self();
    pthread_mutex_unlock(&mu);
    struct timespec t = {0, 300000};  /* time enough for another thread's */
    nanosleep(&t, 0);
    return 0;
}
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int* v, int a, int d) { *v = 256; return 0; }
int hipMalloc(void** p, size_t n) { *p = aligned_alloc(256, 4096); return 0; }  /* never read */
int hipMemsetAsync(void* p, int v, size_t n, void* s) { return 0; }
int hipStreamIsCapturing(void* s, int* c) { *c = 0; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
int hipGetLastError(void) { return 0; }
int launches(void) { return count; }
unsigned long launcher(int i) { return who[i]; }
void forget(void) { count = 0; }
"""

CHILD = r"""
import ctypes, sys, threading, types
stand_in = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # before the library, which then calls it
stand_in.launcher.restype = ctypes.c_ulong
ctypes.CDLL(sys.argv[2])
pkg = types.ModuleType("eredu_amd"); pkg.__path__ = [sys.argv[3] + "/eredu_amd"]  # (without torch)
sys.modules["eredu_amd"] = pkg
from eredu_amd import _native as n
L = n.lib()
P = 1 << 20  # an address that nothing reads
kv = lambda **k: n.KvCache(**{**dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, tables=P, lengths=P, refs=P, missing=P,
    layers=2, pages=100, sequences=8, width=600, kv_heads=8, page_tokens=64, head_dim=128), **k})
caches = [kv(), kv(pages=70000)]
def attend(c, rows, count):
    return lambda: L.eq_kv_attention(P, P, 4096, 32, ctypes.byref(caches[c]), 0, P, count, None, rows, 0.1, True, 0, None, 0, 2, None, 0, None)
CALLS = {
    "attention": attend(0, 3, 3), "attention_rows": attend(1, 300, 1),
    "extend": lambda: L.eq_kv_extend(ctypes.byref(caches[0]), P, 4, None, 1, None, 0, None),
    "extend_many": lambda: L.eq_kv_extend(ctypes.byref(caches[1]), P, 4, None, 1, None, 0, None),
    "fork": lambda: L.eq_kv_fork(ctypes.byref(caches[1]), P, P, 8, None, 0, None),
    "compact": lambda: L.eq_kv_compact(ctypes.byref(caches[0]), None, 0, None),
    "dense_attention": lambda: L.eq_rope_attention_decode(P, P, P, P, P, P, P, 3000, 4096, 32, 8, 128, 0.1, 2, None),
    "matmul": lambda: L.eq_quantized_matmul(P, P, P, P, P, 128, 4096, 4096, True, 64, 4, b"affine", 2, 2, None),
    "matmul_3_bits": lambda: L.eq_quantized_matmul(P, P, P, P, P, 128, 4096, 4096, True, 64, 3, b"affine", 2, 2, None),
    "matmul_not_transposed": lambda: L.eq_quantized_matmul(P, P, P, P, P, 5, 4096, 4096, False, 64, 4, b"affine", 2, 2, None),
    "gguf_linear": lambda: L.eq_gguf_linear(P, P, P, 4096 * 4096 // 256 * 144, 12, 64, 4096, 4096, 0, 2, None),
    "gguf_embedding": lambda: L.eq_gguf_embedding(P, P, 4096 * 4096 // 256 * 144, 12, 4096, 4096, P, 5, 0, 0, None),
    "experts": lambda: L.eq_gather_qmm(P, P, P, P, P, None, P, 512, 512, 8, 1, 1024, 1024, True, 64, 4, b"affine", 2, 2, True, None),
}
names = sys.argv[4].split(",")
each = {}
for name in names:  # alone: how many launches
    stand_in.forget()
    status = CALLS[name]()
    assert status == 0, (name, L.eq_last_error())
    each[name] = stand_in.launches()
    stand_in.forget()
    CALLS[name]()
    assert stand_in.launches() == each[name], name
print(each)
assert all(x > 1 for x in each.values()), each
REPEAT = 12
stand_in.forget()
go = threading.Barrier(len(names))
ids = {}
def work(i):
    ids[threading.get_ident()] = i
    go.wait()
    for _ in range(REPEAT):
        CALLS[names[i]]()
threads = [threading.Thread(target=work, args=(i,)) for i in range(len(names))]
[t.start() for t in threads]; [t.join() for t in threads]
order = [ids[stand_in.launcher(i)] for i in range(stand_in.launches())]
assert len(order) == REPEAT * sum(each[x] for x in names), len(order)
at = switches = 0
while at < len(order):
    mine, n = order[at], each[names[order[at]]]
    assert order[at:at + n] == [mine] * n, (names, at, order[max(0, at - 4):at + 6])
    at += n
    switches += at < len(order) and order[at] != mine
print("switches", switches)
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    d = tmp_path_factory.mktemp("hip")
    src, lib = d / "stand_in.c", d / "libstand_in.so"
    src.write_text(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-w", "-o", str(lib), str(src), "-lpthread"], check=True)
    return str(lib)


@pytest.mark.parametrize("names", ["attention,attention", "attention,attention_rows", "extend,extend_many", "extend,compact",
                                   "fork,attention,extend", "dense_attention,attention", "matmul,attention",
                                   "matmul,matmul_3_bits", "gguf_linear,gguf_embedding,matmul_not_transposed",
                                   "experts,attention,compact"])
def test_launches_of_a_call_stay_together(stand_in, names):
    res = subprocess.run([sys.executable, "-c", CHILD, stand_in, LIB_PATH, ROOT, names], capture_output=True, text=True, timeout=120)
    print(res.stdout)
    assert res.returncode == 0, res.stderr[-2000:]
