"""Launches on arrays of another device than the current one, without a GPU."""

import contextlib

import torch

from flagsparse_amd import _abi


def test_calls_for_another_device_make_it_the_current_one(monkeypatch):
    current = [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        yield
        current[0] = before

    class Library:
        def fsp_anything(self, *args):
            return current[0], args

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_abi, "_lib", Library())
    monkeypatch.setattr(_abi, "_current_device", lambda: current[0])
    monkeypatch.setattr(_abi, "_one_device", False)
    for index, want in ((0, 0), (1, 1), (None, 0)):
        at = torch.device("cuda") if index is None else torch.device("cuda", index)
        assert _abi.lib_on(at).fsp_anything(4, 5) == (want, (4, 5))
        assert current == [0]
    monkeypatch.setattr(_abi, "_one_device", True)
    assert _abi.lib_on(torch.device("cuda", 0)) is _abi.lib()
