"""What a call allocates belongs to the stream that it launches on (no GPU: tensors and library are stand-ins)."""
import contextlib
from types import SimpleNamespace

import pytest
import torch


class _Fake(torch.Tensor):
    """A host tensor that passes for a CUDA one."""
    is_cuda = True


def _fake(t):
    return t.as_subclass(_Fake)


@pytest.fixture
def recorded(monkeypatch):
    """List of (bytes, stream handle) of every allocation; None = the current stream."""
    from smallaios_b200 import ops

    current, seen = [], []

    @contextlib.contextmanager
    def on(stream):
        if stream is None:
            yield
            return
        current.append(stream.cuda_stream)
        yield
        current.pop()

    def allocate(real):
        def call(*a, **kw):
            kw.pop("device", None)
            t = _fake(real(*a, **kw))
            seen.append((t.numel() * t.element_size(), current[-1] if current else None))
            return t
        return call

    def entry(name):
        return lambda *a: 4096 if name.endswith("workspace_bytes") else 0

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda h, device=None: SimpleNamespace(cuda_stream=h))
    for name in ("empty", "empty_like"):
        monkeypatch.setattr(torch, name, allocate(getattr(torch, name)))
    monkeypatch.setattr(ops, "lib", type("Lib", (), {"__getattr__": lambda self, name: entry(name)})())
    monkeypatch.setattr(ops, "_current_stream_handle", lambda device: 0)
    return seen


def _calls(stream):
    from smallaios_b200 import ops

    cache = SimpleNamespace(handle=1, device=torch.device("cpu"), query_width=64, row_shape=(1, 2, 16),
                            tree_workspace_bytes=lambda n, code: 8192)
    q = _fake(torch.zeros(1, 3, 64))
    parents, ids = _fake(torch.zeros(1, 3, dtype=torch.int32)), _fake(torch.zeros(1, 3, 2, 4, dtype=torch.int32))
    means = _fake(torch.zeros(1, 2, 5, 16, dtype=torch.bfloat16))
    ops.gqa_tree_attend(q, cache, 0, parents, num_heads=4, stream=stream)
    ops.gqa_sparse_attend(q, cache, 0, ids, num_heads=4, stream=stream)
    ops.gqa_select_blocks(q, cache, 0, means, num_heads=4, max_blocks=4, stream=stream)
    ops.kv_block_means(cache, 0, 0, 2, stream=stream)


@pytest.mark.parametrize("stream", [SimpleNamespace(cuda_stream=77), 77])
def test_outputs_and_scratch_belong_to_the_launch_stream(recorded, stream):
    _calls(stream)
    assert {n for n, _ in recorded} >= {8192, 4096}  # both workspaces were asked for
    assert {s for _, s in recorded} == {77}


def test_without_a_stream_they_belong_to_the_current_one(recorded):
    _calls(None)
    assert {s for _, s in recorded} == {None}


@pytest.mark.parametrize("host", [True, False])
def test_position_ids_are_made_ready_on_the_launch_stream(recorded, monkeypatch, host):
    """Ids on the host, or strided, are copied by the stream that reads the copy."""
    from smallaios_b200 import ops

    made = []

    class Ids(_Fake):
        is_cuda = not host

        def to(self, *a, **kw):
            torch.empty(1)
            made.append(recorded[-1][1])
            return _fake(self)

        def contiguous(self):
            torch.empty(1)
            made.append(recorded[-1][1])
            return _fake(self)

    monkeypatch.setattr(ops, "_rotary_status_word", lambda device: _fake(torch.zeros(1, dtype=torch.int32)))
    x, table = _fake(torch.zeros(1, 2, 64)), _fake(torch.zeros(4, 8))
    ids = torch.zeros(2, dtype=torch.int32).as_subclass(Ids)
    ops.rotary_embedding(x, table, table, position_ids=ids, num_heads=4, out=x, stream=SimpleNamespace(cuda_stream=77))
    assert made and set(made) == {77}
