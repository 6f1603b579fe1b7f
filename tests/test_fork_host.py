"""A launch in a forked child: torch's own error comes first."""

import os

import torch

from mlx_batch_invariant import _lib


def test_a_forked_child_gets_torch_error(monkeypatch):
    def not_here():
        raise RuntimeError("not in a forked child")

    monkeypatch.setattr(torch.cuda, "_lazy_init", not_here)
    pid = os.fork()
    if pid == 0:
        code = 1
        try:
            _lib.launch_stream(torch.device("cuda", 0))
        except RuntimeError as e:
            code = 0 if "forked child" in str(e) else 2
        finally:
            os._exit(code)
    assert os.waitstatus_to_exitcode(os.waitpid(pid, 0)[1]) == 0
