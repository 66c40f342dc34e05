"""attention_kv8 on a stream that is not the current one, without a GPU: where the memory comes from that the call takes and drops."""
import contextlib
import types

import pytest
import torch

import __graft_entry__ as ge


class OnDevice(torch.Tensor):
    """A host tensor that says it is a device's: what the package's functions look at before they call the library."""
    is_cuda = True


def device_tensor(*shape, dtype):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


class Library:
    """The two entry points, without launches: a workspace is needed, and what was launched is noted."""

    def __init__(self, need):
        self.need, self.calls = need, []

    def ptoamd_attention_kv8_workspace_bytes(self, *args):
        return self.need

    def ptoamd_attention_kv8(self, *args):
        self.calls.append(args)
        return 0


@pytest.mark.parametrize("need", [0, 4096])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("kind", ["torch", "handle"])
def test_a_workspace_is_of_the_stream_that_uses_it(monkeypatch, need, given, kind):
    """The allocator hands a block out again as soon as it is dropped, to work behind what its own stream has: a block of another stream's pool
    would be written by two calls at once."""
    pa = ge.load_package()
    lib, inside, taken = Library(need), [], []
    real_empty = torch.empty

    @contextlib.contextmanager
    def entered(s):
        inside.append(s.cuda_stream)
        yield
        inside.pop()

    def empty(*args, dtype=None, device=None, **kw):
        if dtype == torch.uint8:
            taken.append(inside[-1] if inside else None)
        return real_empty(*args, dtype=dtype, **kw).as_subclass(OnDevice)

    class Stream:
        def __init__(self, handle, device=None):
            self.cuda_stream = handle

    monkeypatch.setattr(pa, "_lib", lib)
    monkeypatch.setattr(torch.cuda, "stream", entered)
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    q = device_tensor(2, 4, 64, dtype=torch.bfloat16)
    codes, scales = device_tensor(4, 2, 16, 64, dtype=torch.int8), device_tensor(4, 2, dtype=torch.float32)
    cache = (codes, codes, scales, scales, device_tensor(2, 2, dtype=torch.int32), device_tensor(2, dtype=torch.int32), pa.I8)
    workspace = {"workspace": device_tensor(4096, dtype=torch.uint8)} if given else {}
    monkeypatch.setattr(torch, "empty", empty)
    stream = Stream(77) if kind == "torch" else types.SimpleNamespace(cuda_stream=77)
    out = pa.attention_kv8.__wrapped__(q, *cache, stream=stream, **workspace) if hasattr(pa.attention_kv8, "__wrapped__") else \
        pa.attention_kv8(q, *cache, stream=stream, **workspace)
    assert out.shape == q.shape and len(lib.calls) == 1 and lib.calls[0][-1] == 77
    assert taken == ([77] if need and not given else [])
