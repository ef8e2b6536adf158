"""Limits of the attention kernels that need no GPU: their tile arithmetic near 32 bits, compiled for
the host."""

import os
import shutil
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "fast_trimul_b200", "csrc")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """Calls a function of the kernels' header with whole numbers, on the host."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    at = tmp_path_factory.mktemp("host")

    def build(name, args):
        src, exe = at / f"{name}.cu", at / name
        if not exe.exists():
            values = ", ".join(f"std::atoi(argv[i + {i}])" for i in range(args))
            src.write_text('#include <cstdio>\n#include <cstdlib>\n#include "ftm_attention.cuh"\n'
                           "int main(int argc, char** argv) {\n"
                           f"  for (int i = 1; i + {args - 1} < argc; i += {args})"
                           f' std::printf("%d\\n", ftm::{name}({values}));\n' "}\n")
            subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr",
                            "-I", CSRC, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                           check=True, capture_output=True)
        return str(exe)

    def call(name, rows):
        exe = build(name, len(rows[0]))
        out = subprocess.run([exe, *[str(x) for r in rows for x in r]], check=True, capture_output=True, text=True)
        return [int(x) for x in out.stdout.split()]

    return call


FAR = [0, 1, 2, 63, 64, 127, 128, 129, 16_777_216, 16_777_217, 17_000_000, 33_554_432, 2 ** 30, 2 ** 31 - 1024]


def test_columns_in_front_of_the_first_query(host):
    rows = [(s * n, g) for n in FAR for s in (1, -1) for g in (1, 2, 3, 64, 127, 128)]
    assert host("columns_before", rows) == [max(0, min(128, a * g)) for a, g in rows]


def test_rows_of_a_query_tile(host):
    rows = [(n, 128 // g, g) for n in FAR[1:] for g in (1, 2, 3, 64, 127, 128)]
    assert host("rows_held", rows) == [min(n, tq) * g for n, tq, g in rows]


def test_lengths_past_32_bits_are_clamped_not_wrapped():
    import torch
    from fast_trimul_b200.functional import cached_attention
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(*s, generator=g) for s in ((5, 4, 8), (5, 9, 2, 8), (5, 9, 2, 8)))
    got = cached_attention(q, k, v, torch.tensor([2 ** 31, 2 ** 32 + 3, 2 ** 62, -2 ** 32 + 4, 7]))
    want = cached_attention(q, k, v, torch.tensor([9, 9, 9, 0, 7], dtype=torch.int32))
    assert torch.equal(got, want)
    got = cached_attention(q, k, v, torch.tensor([2 ** 31, 9, 9, 0, 7], dtype=torch.uint32))
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        cached_attention(q, k, v, torch.ones(5, dtype=torch.complex64))


# ------------------------------------------------------------------- failures and several threads
class Calls:
    """Runs calls in a thread of its own, one after the other."""

    def __init__(self):
        import concurrent.futures
        self.pool = concurrent.futures.ThreadPoolExecutor(max_workers=1)

    def __call__(self, f):
        return self.pool.submit(f).result()


@pytest.fixture
def error_word(monkeypatch):
    """An AttentionErrorWord without a GPU, and what it does: "synchronize", "zero", "clear" and "count"
    in order."""
    import torch
    from fast_trimul_b200.ops.attention import AttentionErrorWord
    done = []

    class Dev:
        device = torch.device("cuda", 63)

        def zero_(self):
            done.append("zero")

    class Word:
        now = 0

        @property
        def value(self):
            return self.now

        @value.setter
        def value(self, x):
            if x == 0:
                done.append("clear")
            self.now = x

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: done.append("synchronize"))
    w = AttentionErrorWord.__new__(AttentionErrorWord)
    import threading
    w.dev, w.word, w.index, w.code, w.lock = Dev(), Word(), 63, 0, threading.Lock()
    return w, done


def test_every_thread_that_called_learns_of_a_failure_once(error_word):
    """Kernels of all streams give up together: who polls first must not be the only one to hear of it."""
    from fast_trimul_b200 import _lib
    w, _ = error_word
    a, b, late = Calls(), Calls(), Calls()
    a(w.poll)                    # each has called before ...
    b(w.poll)
    w.word.now = 0x421           # ... a wait expires ...
    for thread in (a, b):
        with pytest.raises(_lib.NativeKernelError, match="0x421"):
            thread(w.poll)
        thread(w.poll)           # ... and each hears of it once
    late(w.poll)                 # a thread that had nothing running hears nothing
    w.word.now = 0x512
    with pytest.raises(_lib.NativeKernelError, match="0x512"):
        late(w.poll)
    for thread in (a, b):
        with pytest.raises(_lib.NativeKernelError, match="0x512"):
            thread(w.poll)
    fresh = Calls()              # one whose first call finds the word set hears of it, too
    w.word.now = 0x631
    with pytest.raises(_lib.NativeKernelError, match="0x631"):
        fresh(w.poll)


def test_the_host_word_is_cleared_last(error_word):
    """While the device word may still be set, launches of other threads have to find the host word set."""
    from fast_trimul_b200 import _lib
    w, done = error_word
    w.word.now = 0x421
    with pytest.raises(_lib.NativeKernelError):
        w.poll()
    assert done == ["synchronize", "zero", "synchronize", "clear"] and w.word.now == 0


def test_large_batches_of_a_cache_are_not_refused():
    """Items of a cache are its tiles times heads times sequences: sequences were counted twice, and 16 384
    sequences of 8 heads refused; and a product past 64 bits must not wrap to a small one."""
    from fast_trimul_b200 import _lib
    lib, p = _lib.load(), 1 << 20

    def taken(sequences, heads, capacity):
        a = _lib.Attention(dtype=_lib.BF16, heads=heads, kv_heads=heads, head_dim=64, scale=0.125, sequences=sequences,
                           q_len=1, q_rows=sequences, kv_rows=capacity, kv_lengths=p, q=p, q_row_stride=64 * heads,
                           q_head_stride=64, k=p, k_row_stride=64 * heads, k_head_stride=64,
                           k_batch_stride=64 * heads * capacity, v=p, v_row_stride=64 * heads, v_head_stride=64,
                           v_batch_stride=64 * heads * capacity, out=p)
        return lib.ftm_attention_workspace_bytes(a, 0) > 0      # 0: refused

    assert taken(16, 8, 16384) and taken(16384, 8, 4096) and taken(6000, 64, 512)
    assert not taken(1 << 20, 64, 4096)                         # 2^31 items
    assert not taken(2 ** 31 - 2048, 1 << 30, 256)
