"""The Python binding of the quantised paged KV cache without a GPU: what it hands to the C calls, and its refusals."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on cuda:0 (no call here reaches a device)."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32).as_subclass(OnGpu)


def test_a_slice_of_a_table_bounds_its_sequences(nb):
    """Four columns of a table of sixteen: 64 tokens of 16 a sequence, not 256."""
    table = torch.zeros((3, 16), dtype=torch.int32)[:, 12:].as_subclass(OnGpu)
    batch = nb.KvBatch(i32(4), i32(3), table, 1, 200)
    t = batch._ref(0, 16)._obj
    assert (t.n_seqs, t.table_stride, t.max_kv) == (3, 16, 64)
    assert batch._ref(0, 64)._obj.max_kv == 200  # pages of 64 tokens hold 256
    assert batch._ref(0, 16)._obj.max_kv == 64
    assert batch.max_kv == 200


def test_the_package_needs_no_torch_until_the_cache_is_used():
    """A star import without torch works; the names of the paged cache ask for it."""
    code = """
import sys
sys.modules["torch"] = None   # import torch raises ImportError
from nexus_b200 import *
CudaBackend, Scheduler
import nexus_b200
try:
    nexus_b200.PagedKvCache
except ImportError:
    print("asked")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "asked\n", r.stderr


def test_the_paged_cache_is_a_name_of_the_package(nb):
    from nexus_b200 import KvBatch, PagedKvCache
    assert nb.KvBatch is KvBatch and nb.PagedKvCache is PagedKvCache


def test_a_batch_is_of_its_tensors_and_bounds_for_good(nb):
    """The struct handed to the calls holds their addresses: another tensor is another batch."""
    batch = nb.KvBatch(i32(4), i32(3), i32(3, 8), 2, 100)
    kept = batch.kv_len
    for name, value in (("q_start", i32(4)), ("kv_len", i32(3)), ("page_table", i32(3, 8)), ("max_q", 3), ("max_kv", 9)):
        with pytest.raises(AttributeError):
            setattr(batch, name, value)
    t = batch._ref(0, 16)._obj
    assert batch.kv_len is kept and t.kv_len == kept.data_ptr() and (t.max_q, t.max_kv) == (2, 100)


def test_what_a_batch_keeps_is_bounded(nb):
    batch = nb.KvBatch(i32(4), i32(3), i32(3, 8), 2, 100)
    for stream in range(1, 1000):
        t = batch._ref(stream, 16)._obj
        assert t.stream == stream
    assert len(batch._structs) <= 64


@pytest.mark.parametrize("value", [-1, 2 ** 31, 2 ** 32, 2 ** 32 + 5])
@pytest.mark.parametrize("name", ["window", "sinks"])
def test_window_and_sinks_beyond_32_bits_are_refused(nb, name, value):
    """2^32 is not a window of 0, which would see the whole context."""
    c = nb.PagedKvCache.__new__(nb.PagedKvCache)
    with pytest.raises(nb.NexusError, match="window and sinks"):
        c.attention(None, None, **{name: value})


def test_rows_that_require_a_gradient_are_refused(nb):
    """There is no backward pass; a result without history would drop the gradient silently."""
    c = nb.PagedKvCache.__new__(nb.PagedKvCache)
    x = torch.zeros((2, 4, 64), requires_grad=True)
    for call in (lambda: c.attention(None, x), lambda: c.append(None, x, x.detach()),
                 lambda: c.append(None, x.detach(), x)):
        with pytest.raises(nb.NexusError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(AttributeError):  # past the check, on to the (missing) batch
            call()


def test_the_binding_needs_torchs_public_interface_only():
    """A torch without the private lookup of the current stream: torch.cuda.current_stream serves."""
    code = """
import torch
from types import SimpleNamespace
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    del torch._C._cuda_getCurrentRawStream
torch.cuda.current_stream = lambda device: SimpleNamespace(cuda_stream=1234 + device)
from nexus_b200 import paged
print(paged._raw_stream(1))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "1235\n", r.stderr
