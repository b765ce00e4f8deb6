"""The Python side of the paged-cache calls without a GPU: a library that only notes its arguments, and tensors that say
they are on a GPU."""
import contextlib

import pytest
import torch

from metalqwen3_b200 import q3cu


class Tensor:
    """What the binding asks of a tensor."""

    def __init__(self, shape, dtype=torch.bfloat16, device=0, made_on=None):
        self.t = torch.empty(shape, dtype=dtype)
        self.shape, self.dtype, self.made_on, self.used_on = self.t.shape, dtype, made_on, []
        self.index, self.device, self.is_cuda = device, "cpu" if device < 0 else f"cuda:{device}", device >= 0
        self.nbytes = self.t.nbytes

    def get_device(self):
        return self.index

    def record_stream(self, stream):
        self.used_on.append(stream)

    def new_empty(self, *a):
        return self.t.new_empty(*a)

    def __getattr__(self, name):                             # stride, dim, numel, data_ptr, is_contiguous ...
        return getattr(self.t, name)


class Library:
    """Notes the calls and says that all is well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            if name == "q3cu_attention_paged_workspace":
                args[-1]._obj.value = 64
            return 0
        return call


class Stream:
    def __init__(self, name):
        self.cuda_stream = self.name = name


@pytest.fixture
def binding():
    q = q3cu.Q3CU.__new__(q3cu.Q3CU)
    main = Stream(7)

    class Cuda:
        current, Stream = main, Stream

        @staticmethod
        def ExternalStream(handle, device):
            return Stream(handle)

        @contextlib.contextmanager
        def stream(self, s):
            before, self.current = self.current, s
            yield
            self.current = before

        def current_stream(self, device=None):
            return self.current

    class Torch:
        cuda, uint8, float32 = Cuda(), torch.uint8, torch.float32
        made = []

        def empty(self, shape, dtype, device):
            self.made.append(Tensor(shape, dtype, int(device[-1]), self.cuda.current))
            return self.made[-1]

    q.torch, q.lib, q.device, q.ctx, q._raw_stream = Torch(), Library(), 0, None, None
    q.torch.made = []
    q.main = main
    return q


def cache_and_batch(device=0):
    k, v = (Tensor((4, 2, 16, 128), device=device) for _ in range(2))
    i32 = torch.int32
    return q3cu.KVCache(k, v), q3cu.KVBatch(Tensor((3,), i32, device), Tensor((3, 2), i32, device), Tensor((4,), i32, device))


@pytest.mark.parametrize("given", [False, True])
def test_calls_make_their_memory_on_their_stream(binding, given):
    """Results and workspaces come from the memory of the stream that uses them; what the caller gets is also marked as
    used on the current one."""
    stream = Stream(9) if given else None
    on = stream or binding.main
    cache, batch = cache_and_batch()
    q, k = Tensor((3, 4, 128)), Tensor((3, 2, 128))
    results = [binding.kv_append(cache, batch, q, k, k, stream=stream), binding.attention_paged(cache, batch, q, stream=stream),
               binding.attention_prompt(cache, batch, q, stream=stream)]
    assert len(binding.torch.made) == 4 and all(t.made_on is on for t in binding.torch.made)
    assert binding.torch.cuda.current is binding.main
    if given:
        assert all(binding.main in t.used_on for t in results)
    assert {args[-1] for name, args in binding.lib.calls if "workspace" not in name} == {on.cuda_stream}
    if given:
        assert binding.attention_paged_workspace(cache, 4, stream=stream).made_on is on


def test_a_stream_known_by_its_handle(binding):
    """What has a stream's handle and nothing else of torch's streams."""
    class Handle:
        cuda_stream = 11

    cache, batch = cache_and_batch()
    binding.attention_paged(cache, batch, Tensor((3, 4, 128)), stream=Handle())
    assert [t.made_on.cuda_stream for t in binding.torch.made] == [11, 11]


def test_memory_elsewhere_is_refused(binding):
    """A cache, a batch or a workspace on another GPU or on the host, or a workspace that is not all there, reaches no
    kernel."""
    cache, batch = cache_and_batch()
    far_cache, far_batch = cache_and_batch(1)
    q, k = Tensor((3, 4, 128)), Tensor((3, 2, 128))
    for c, b in ((far_cache, batch), (cache, far_batch)):
        for call in (lambda: binding.kv_append(c, b, q, k, k), lambda: binding.attention_paged(c, b, q),
                     lambda: binding.attention_prompt(c, b, q)):
            with pytest.raises(ValueError, match="must be on the context's GPU"):
                call()
    spread = Tensor((1,), torch.uint8)
    spread.t, spread.nbytes = spread.t.expand(1 << 20), 1 << 20
    for work in (Tensor((1 << 20,), torch.uint8, -1), Tensor((1 << 20,), torch.uint8, 1), spread):
        with pytest.raises(ValueError, match="work must be contiguous memory on the context's GPU"):
            binding.attention_paged(cache, batch, q, work=work)
    assert not binding.lib.calls
    i32 = torch.int32
    for pages, row_off in ((1, 0), (0, 1), (0, -1)):
        with pytest.raises(ValueError, match="must be on the context's GPU"):
            q3cu.KVBatch(Tensor((3,), i32), Tensor((3, 2), i32, pages), Tensor((4,), i32, row_off))
    binding.attention_paged(cache, batch, q, work=Tensor((1 << 20,), torch.uint8))
    assert binding.lib.calls
