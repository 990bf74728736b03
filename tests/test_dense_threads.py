"""Python threads that enqueue through one context, or through contexts that share workspaces, take turns: the arrays that a call is
given reach the library together, and no other call's launches come between those of one call. And a call may be the first thing
that a thread does with the GPU."""
import contextlib
import ctypes
import threading
import time

import pytest
import torch

import hashattention_b200 as ha
from hashattention_b200 import _lib, dense, synthetic
from test_dense import D, Problem

T = 4


class FakeLibrary:
    """Records what every call finds in its structs after another thread has had the time to change them."""

    def __init__(self):
        self.seen, self.running, self.together = [], 0, 0

    def _call(self, name, tree, *rest):
        self.running += 1
        self.together = max(self.together, self.running)
        time.sleep(0.02)  # (the interpreter is released, as in a call through ctypes)
        self.seen.append((name, tree.max_nodes, tree.tree_mask, tree.tree_lens) + rest)
        self.running -= 1
        return _lib.HA_OK

    def ha_tree_attention(self, shape, tree, q, strides, *rest):
        return self._call("attention", tree, q, tuple(strides))

    def ha_attention_mass(self, shape, tree, q, strides, *rest):
        return self._call("mass", tree, q, tuple(strides))

    def ha_tree_commit(self, shape, tree, accepted, *rest):
        return self._call("commit", tree, accepted)

    def ha_cache_evict(self, *args):
        return self._call("evict", _lib.HaTree(0, None, None))


def context(lib, share=None):
    """A context on CPU tensors with a library that launches nothing."""
    ctx = object.__new__(ha.DenseDecodeContext)
    ctx.__dict__.update(
        lib=lib, cache=ha.PagedHashKVCache(1, 1, 256, "cpu"), device=torch.device("cpu"), max_nodes=T, batch=1, num_kv_heads=1,
        num_q_heads=4, sm_scale=1.0, shape=_lib.HaShape(1, 1, 4, 128, 256, 1, 1, 1), _shape_ref=None, workspace_bytes=8,
        evict_workspace_bytes=8, status=torch.zeros(1, dtype=torch.int32), _workspace_ptr=0, _evict_workspace_ptr=0, _status_ptr=0,
        _c_tree=_lib.HaTree(), _c_strides=(ctypes.c_int64 * 3)(), _turn=threading.Lock() if share is None else share._turn)
    return ctx


def run_threads(jobs):
    start = threading.Barrier(len(jobs))
    errors = []

    def body(job):
        try:
            start.wait(10)
            job()
        except Exception as e:  # (a failure belongs to the test, not to the thread)
            errors.append(e)

    threads = [threading.Thread(target=body, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert not errors, errors


def jobs_for(ctx, count):
    """Calls of every kind with arrays of their own -> (jobs, what the library has to see)."""
    jobs, want = [], []
    for i in range(count):
        n = 1 + i % T
        q = torch.zeros(1, n, 4 + i, 128, dtype=torch.bfloat16)[:, :, :4]
        mask, lens = torch.zeros(1, n, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
        lse, mass = torch.zeros(1, n, 4), torch.zeros(1, 1, 256)
        strides = (0, 0 if n == 1 else q.stride(1), 128)
        jobs.append(lambda q=q, mask=mask, lens=lens: ctx.tree_attention(q, mask, lens))
        want.append(("attention", n, mask.data_ptr(), lens.data_ptr(), q.data_ptr(), strides))
        jobs.append(lambda q=q, mask=mask, lse=lse, mass=mass: ctx.attention_mass(q, lse, mass, mask))
        want.append(("mass", n, mask.data_ptr(), None, q.data_ptr(), strides))
        accepted = torch.zeros(1, 4, dtype=torch.int32)
        jobs.append(lambda accepted=accepted, lens=lens: ctx.tree_commit(accepted, lens))
        want.append(("commit", T, None, lens.data_ptr(), accepted.data_ptr()))
        jobs.append(lambda mass=mass: ctx.cache_evict(mass, 8, 1, 1))
        want.append(("evict", 0, None, None))
    return jobs, want


def test_threads_on_one_context_take_turns(monkeypatch):
    monkeypatch.setattr(dense, "library_call", lambda device, name: contextlib.nullcontext())
    monkeypatch.setattr(dense, "_stream_ptr", lambda device: 0)
    lib = FakeLibrary()
    jobs, want = jobs_for(context(lib), 4)
    run_threads(jobs)
    assert sorted(map(str, lib.seen)) == sorted(map(str, want))
    assert lib.together == 1


def test_threads_on_contexts_that_share_a_workspace_take_turns(monkeypatch):
    monkeypatch.setattr(dense, "library_call", lambda device, name: contextlib.nullcontext())
    monkeypatch.setattr(dense, "_stream_ptr", lambda device: 0)
    lib = FakeLibrary()
    first = context(lib)
    more, want = jobs_for(context(lib, share=first), 2)
    jobs, want_first = jobs_for(first, 2)
    run_threads(jobs + more)
    assert sorted(map(str, lib.seen)) == sorted(map(str, want + want_first))
    assert lib.together == 1


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["attention of 1 node", "attention of 6 nodes", "received weights", "key hashes", "eviction", "commit"])
def test_the_first_cuda_call_of_a_thread(device, call):
    """A new thread has no CUDA context of its own until the runtime gives it one: the library's entry points must not need it before."""
    n = 1 if call == "attention of 1 node" else 6
    x = Problem(device, [700, 300], [n, n], 2, n, "chain", seed=1)
    out, lse = x.ctx.tree_attention(x.q)
    mass, want = x.ctx.new_mass(), x.ctx.attention_mass(x.q, lse, x.ctx.new_mass())
    sparse = ha.SparseDecodeContext(x.cache, ha.Budget(8, 0.25, 8), synthetic.make_usa(8, D, seed=0, bf16=True).packed(device))
    sparse.hash_prefill()
    codes = x.cache.hash_pages.clone()
    o2, l2 = torch.zeros_like(out), torch.zeros_like(lse)
    words, rest = torch.zeros(2, 4, dtype=torch.int32, device=device), x.ctx.cache_evict(mass, 1000, 4, 4)
    kept = rest[0].clone()
    torch.cuda.synchronize()
    run_threads([{"attention of 1 node": lambda: x.ctx.tree_attention(x.q, out=o2, lse=l2),
                  "attention of 6 nodes": lambda: x.ctx.tree_attention(x.q, out=o2, lse=l2),
                  "received weights": lambda: x.ctx.attention_mass(x.q, lse, mass),
                  "key hashes": sparse.hash_prefill,
                  "eviction": lambda: x.ctx.cache_evict(mass, 1000, 4, 4, kept=rest[0], mass_out=rest[1], lens_out=rest[2]),
                  "commit": lambda: x.ctx.tree_commit(words, max_nodes=n)}[call]])
    x.ctx.check_status()
    if call.startswith("attention"):
        assert torch.equal(o2, out) and torch.equal(l2, lse)
    if call == "received weights":
        assert torch.equal(mass, want)
    assert torch.equal(x.cache.hash_pages, codes) and torch.equal(rest[0], kept)
