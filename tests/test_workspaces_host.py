"""The workspaces that calls of a thread share, on the CPU: they go with their
thread, and stay with the others."""

import subprocess
import sys
import threading
import weakref

import pytest
import torch

from dropkv_amd import ops

DEV = torch.device("cuda", 0)


class Workspace:
    """In place of a tensor: its release can be watched."""

    def __init__(self, nbytes):
        self.nbytes = nbytes

    def numel(self):
        return self.nbytes


@pytest.fixture
def made(monkeypatch):
    """Weak references to the workspaces made."""
    refs = []

    def make(nbytes, dev):
        ws = Workspace(nbytes)
        refs.append(weakref.ref(ws))
        return ws

    monkeypatch.setattr(ops, "_shared_ws", {})
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_evict_workspace", make)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return refs


def test_an_ended_thread_keeps_nothing(made):
    """One after another, forty threads with a workspace each, some grown: what
    is held at the end is this thread's."""
    mine = ops._stream_workspace(100, DEV)

    def call():
        ops._stream_workspace(1000, DEV)
        ops._stream_workspace(2000, DEV)

    for _ in range(40):
        t = threading.Thread(target=call)
        t.start()
        t.join()
    assert [r() for r in made if r() is not None] == [mine]
    assert list(ops._shared_ws.values()) == [mine] and ops._stream_workspace(100, DEV) is mine


def test_threads_at_work_keep_theirs(made):
    """While other threads end, a thread's workspace stays its own; afterwards
    release_workspaces still reaches every thread's."""
    done, go_on = threading.Event(), threading.Event()
    seen = []

    def stay():
        seen.append(ops._stream_workspace(500, DEV))
        done.set()
        go_on.wait(30)
        seen.append(ops._stream_workspace(500, DEV))
        ops.release_workspaces()
        seen.append(ops._stream_workspace(500, DEV))

    worker = threading.Thread(target=stay)
    worker.start()
    assert done.wait(30)
    for _ in range(3):
        t = threading.Thread(target=ops._stream_workspace, args=(700, DEV))
        t.start()
        t.join()
    mine = ops._stream_workspace(100, DEV)
    go_on.set()
    worker.join()
    assert seen[0] is seen[1] and seen[2] is not seen[0]
    assert not ops._shared_ws
    assert ops._stream_workspace(100, DEV) is not mine


def test_the_end_of_the_interpreter():
    """A workspace of the main thread's at the end of the process: no complaint."""
    code = ("import torch\n"
            "from dropkv_amd import ops\n"
            "ops._stream = lambda dev: 0\n"
            "ops._evict_workspace = lambda nbytes, dev: torch.zeros(nbytes)\n"
            "torch.cuda.is_current_stream_capturing = lambda: False\n"
            "ops._stream_workspace(10, torch.device('cuda', 0))\n")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "Exception" not in run.stderr, run.stderr
