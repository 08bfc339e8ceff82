"""The training calls leave the caller's current device as it was."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "device_scope.h"
static int current = 0, sets = 0, fail_get = 0, fail_set = -1;
struct Fake {
  static int get(int* d) { *d = current; return fail_get; }
  static int set(int d) { ++sets; if (d == fail_set) return 101; current = d; return 0; }
};
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  using Scope = tessa::DeviceScope<Fake>;
  for (int from = 0; from < 3; ++from)
    for (int to = 0; to < 3; ++to) {
      current = from;
      {
        Scope s;
        CHECK(s.enter(to) == 0 && current == to);
      }
      CHECK(current == from);
    }
  current = 1;
  sets = 0;
  { Scope never; }
  CHECK(sets == 0);
  fail_set = 2;
  {
    Scope s;
    CHECK(s.enter(2) == 101);
  }
  CHECK(current == 1);
  fail_get = 3;
  {
    Scope s;
    CHECK(s.enter(0) == 3 && current == 1);
  }
  CHECK(current == 1);
  return 0;
}
"""


def test_the_scope_puts_the_device_back(tmp_path):
    src, exe = tmp_path / "scope.cpp", tmp_path / "scope"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{ROOT}/shear_b200/csrc", str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_every_training_call_keeps_to_it():
    # (where there is one GPU, nothing else shows it): each begins through async_begin, which enters a scope
    import re
    with open(os.path.join(ROOT, "shear_b200", "csrc", "capi_train.cu")) as f:
        train = f.read()
    with open(os.path.join(ROOT, "shear_b200", "csrc", "capi.cu")) as f:
        capi = f.read()
    assert "cudaSetDevice" not in train and "bind(" not in train
    assert train.count("TRY(async_begin(ctx, &c));") == 5
    # the last reference to a context may go anywhere
    for name in ("tessa::async_begin", "tessa_async_status", "tessa_destroy"):
        body = re.search(rf"(?:int|void) {name}\(.*?\n}}\n", capi, re.S).group(0)
        assert "scope" in body and "bind(" not in body and "cudaSetDevice" not in body, name


def test_a_context_made_by_a_training_call(monkeypatch):
    # in Python, as the C call that makes one leaves its device current
    import contextlib
    import threading

    import torch
    from shear_b200 import ops
    current = [0]

    @contextlib.contextmanager
    def device(i):
        before, current[0] = current[0], i
        yield
        current[0] = before

    class Fake:
        def __init__(self, dev):
            current[0] = self.device = dev

    ops._lazy_torch()
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(ops, "Context", Fake)
    monkeypatch.setattr(ops, "_tls", threading.local())
    made = ops._context(1)
    assert made.device == 1 and current == [0]
    assert ops._context(1) is made is ops.context(1) and ops._context(0) is not made and current == [0]


@pytest.mark.gpu
def test_a_call_on_another_device():
    import torch
    from shear_b200 import ops
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    table, ids = torch.randn(9, 8, device="cuda:1"), torch.arange(4, device="cuda:1")
    torch.cuda.set_device(0)
    got = ops.embedding_lookup(table, ids)  # makes the thread's context
    assert torch.cuda.current_device() == 0
    ops.async_status(device=1)
    assert torch.cuda.current_device() == 0 and torch.equal(got, table[:4])
