"""CUDA calls that fail in the middle of a tree pass.  The failures are made on
the host: a preloaded library answers for one call of the runtime with an error
code, and nothing reaches the device that would not otherwise."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

HERE = Path(__file__).resolve().parent
FAKE = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <stddef.h>
#include <string.h>

static int event_in, copy_in, syncs_after;  /* calls until one fails: 0 none */
static size_t copy_bytes;
void fake_event(int in) { event_in = in; syncs_after = -1; }
void fake_copy(int in, size_t bytes) { copy_in = in, copy_bytes = bytes; syncs_after = -1; }
int fake_syncs(void) { return syncs_after; }  /* since the call that failed; -1: none failed */
static void* real(const char* name) {  /* the runtime that the engine's library brought along */
    static void* lib;
    if (!lib) lib = dlopen("libcudart.so.12", RTLD_LAZY | RTLD_NOLOAD);
    return dlsym(lib, name);
}

int cudaEventRecord(void* e, void* s) {
    if (event_in && !--event_in) { syncs_after = 0; return 999; }
    return ((int (*)(void*, void*))real("cudaEventRecord"))(e, s);
}
int cudaMemcpyAsync(void* d, const void* s, size_t n, int kind, void* st) {
    if (copy_in && (!copy_bytes || copy_bytes == n) && !--copy_in) { syncs_after = 0; return 999; }
    return ((int (*)(void*, const void*, size_t, int, void*))real("cudaMemcpyAsync"))(d, s, n, kind, st);
}
int cudaStreamSynchronize(void* s) {
    if (syncs_after >= 0) ++syncs_after;
    return ((int (*)(void*))real("cudaStreamSynchronize"))(s);
}
"""

HEAD = """
import ctypes, os, sys
sys.path[:0] = {paths!r}
import numpy as np
import jalapeno as J
import oracle as O
import dataclasses
fake = ctypes.CDLL({so!r})
fake.fake_copy.argtypes = [ctypes.c_int, ctypes.c_size_t]
cfg = dataclasses.replace(O.PRESETS["tiny"], name="tiny-q8-kv2", q_heads=8, kv_heads=2, max_positions=1024)
m = J.Model.from_config(cfg, 3, mxfp4=True)
"""


def child(tmp_path, body):
    src, so = tmp_path / "fake.c", tmp_path / "fake.so"
    src.write_text(FAKE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", str(so), str(src), "-ldl"], check=True)
    code = HEAD.format(paths=[p for p in sys.path if p], so=str(so)) + body
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, LD_PRELOAD=str(so)))
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_a_failed_tree_pass_waits_for_what_it_queued(tmp_path):
    """The event after the descriptors' copies, and the copy of the logits after
    the ids': the call reports the error once nothing is in flight, keeps no tree,
    and the next one is right."""
    child(tmp_path, """
c = m.cache()
m.predict(O.prompt_ids(70, cfg.vocab, 5), c)
tokens, parents = O.prompt_ids(5, cfg.vocab, 6), [-1, 0, 0, 1, 2]
want, wlg = m.predict_tree(tokens, parents, c, logits=True)
for arm in (lambda: fake.fake_event(1), lambda: fake.fake_copy(1, 5 * cfg.vocab * 4), lambda: fake.fake_copy(5, 0)):
    arm()
    try:
        m.predict_tree(tokens, parents, c, logits=True)
        raise SystemExit("no error")
    except J.JlError as e:
        assert e.status == J.JL_ERR_CUDA, e
    assert fake.fake_syncs() > 0, "returned with work in flight"
    try:
        c.compact([0])
        raise SystemExit("a tree was kept")
    except J.JlError:
        pass
    assert c.len == 70
    ids, lg = m.predict_tree(tokens, parents, c, logits=True)
    assert ids == want and np.array_equal(lg, wlg)
print("ok")
""")


def test_a_failed_unsharing_leaves_the_fork_alone(tmp_path):
    """The copy of a new page's table entry: after the error the cache still
    holds the shared page, and its next write copies it first."""
    child(tmp_path, """
prompt = O.prompt_ids(128, cfg.vocab, 5)
a, c = m.cache(), m.cache()
m.predict(prompt, a)
m.predict(prompt, c)
f = a.fork()
a.truncate(70)
fake.fake_copy(1, 4)
try:
    m.predict(O.prompt_ids(40, cfg.vocab, 8), a)
    raise SystemExit("no error")
except J.JlError as e:
    assert e.status == J.JL_ERR_CUDA, e
assert a.len == 70
m.predict(O.prompt_ids(40, cfg.vocab, 8), a)
for t in (1, 2):
    assert np.array_equal(m.predict([t], f, logits=True)[1], m.predict([t], c, logits=True)[1])
g = m.cache()
m.predict(prompt[:70], g)
m.predict(O.prompt_ids(40, cfg.vocab, 8), g)
assert np.array_equal(m.predict([9], a, logits=True)[1], m.predict([9], g, logits=True)[1])
print("ok")
""")
