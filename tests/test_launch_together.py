"""A call holds its workspace's lock while it queues its kernels, so that none of another thread's comes between them.

Which mutexes a call takes is recorded by a `pthread_mutex_lock` in front of the C library's, in a process without a device: the calls
come as far as their first CUDA call, with the lock held.  The workspace's lock is the one that changes with the workspace."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest

from fhob import _lib

RECORDER = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <pthread.h>
static void* taken[4096];
static int count, recording;
int pthread_mutex_lock(pthread_mutex_t* m) {
  static int (*next)(pthread_mutex_t*);
  if (!next) next = (int (*)(pthread_mutex_t*))dlsym(RTLD_NEXT, "pthread_mutex_lock");
  if (recording && count < 4096) taken[count++] = m;
  return next(m);
}
void record(int on) { recording = on; if (on) count = 0; }
int recorded(void** to) { for (int i = 0; i < count; ++i) to[i] = taken[i]; return count; }
"""

CHILD = r"""
import ctypes as C, sys
from fhob import _lib
recorder, lib = C.CDLL(sys.argv[1]), _lib.load()

def locks(call, workspace, sinks, n_q, dtype):
    p = _lib.FhobProblem()
    p.bh, p.n_q, p.n_k, p.d, p.dtype, p.causal, p.window = 1, n_q, 300, 64, dtype, 1, 20
    for n in ("q", "k", "v", "o", "d_o", "ddq", "ddk", "ddv", "lse", "dq2", "dk2", "dv2", "ddo"):
        setattr(p, n, 4096)
    p.workspace, p.workspace_bytes = workspace, 1 << 22
    recorder.record(1)
    status = call(C.byref(p), sinks)
    recorder.record(0)
    assert status in (5, 6), status      # no device: a CUDA call failed, or there is none of the architecture
    got = (C.c_void_p * 4096)()
    return set(got[:recorder.recorded(got)])

calls = {
    "forward": lambda p, s: lib.fhob_forward_sinks(p, s, 4096, 4096, None),
    "backward": lambda p, s: lib.fhob_backward_sinks(p, s, 4096, 4096, 4096, None),
    "operator": lambda p, s: lib.fhob_bwdbwd_sinks(p, s, None),
}
here, there = 1 << 20, (1 << 20) + (5 << 8)
for name, call in calls.items():
    call_locks = lambda w, s, n, t: locks(call, w, s, n, t)
    for sinks in (0, 4):
        for n_q in (1, 2, 3, 200):
            for dtype in (0, 1, 2):
                call_locks(here, sinks, n_q, dtype)      # (what is set up once)
                a, b = call_locks(here, sinks, n_q, dtype), call_locks(there, sinks, n_q, dtype)
                assert len(a - b) == 1 and len(b - a) == 1, (name, sinks, n_q, dtype, len(a - b), len(b - a))
print("ok")
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no gcc")
def test_every_call_takes_its_workspaces_lock(tmp_path):
    (tmp_path / "recorder.c").write_text(RECORDER)
    shim = tmp_path / "recorder.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", str(shim), str(tmp_path / "recorder.c"), "-ldl"], check=True)
    env = dict(os.environ, LD_PRELOAD=str(shim), CUDA_VISIBLE_DEVICES="", PYTHONPATH=os.path.dirname(os.path.dirname(_lib.__file__)))
    r = subprocess.run([sys.executable, "-c", CHILD, str(shim)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
