"""Where the tensors of the 8-bit cache's and the sampling bindings may be, and their shapes.  No GPU and no launch: the
tensors are on the host, get_device() says what the test wants, and the library is a stand-in that counts its calls."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

I32 = torch.int32


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith("workspace_size"):
            return lambda *a: 256

        def entry(*a):
            self.calls.append(name)
            return 0

        return entry


@pytest.fixture
def world(monkeypatch):
    """(ops, library, places): places maps a tensor's address to its device, 0 where it is absent."""
    from onnxruntime_ep_b200 import ops

    ops._lib()
    library, places = Library(), {}
    monkeypatch.setattr(ops, "_lib", lambda: library)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: places.get(t.data_ptr(), 0))
    return ops, library, places


def cache():
    codes = [torch.zeros(4, 2, 8, 64, dtype=torch.int8) for _ in range(2)]
    return dict(key_cache=codes[0], value_cache=codes[1], key_scales=torch.zeros(4, 2, 8), value_scales=torch.zeros(4, 2, 8))


def tables():
    return dict(cumulative_seqlens=torch.tensor([0, 1, 2], dtype=I32), past_seqlens=torch.zeros(2, dtype=I32),
                block_table=torch.zeros(2, 2, dtype=I32), cos_cache=torch.zeros(9, 32).half(),
                sin_cache=torch.zeros(9, 32).half())


def rows(*heads):
    return [torch.zeros(2, n * 64).half() for n in heads]


def arguments(name):
    if name == "paged_kv_quantize":
        return dict(zip(("key", "value"), rows(2, 2)), **cache(), **tables()), {}
    if name == "paged_kv_dequantize":
        return dict(cache(), seqlens=torch.zeros(2, dtype=I32), block_table=torch.zeros(2, 2, dtype=I32),
                    key=torch.zeros(2, 2, 5, 64).half(), value=torch.zeros(2, 2, 5, 64).half()), {}
    if name == "paged_attention_quantized":
        q, k, v, out = rows(4, 2, 2, 4)
        return dict(cache(), query=q, key=k, value=v, out=out, workspace=torch.zeros(256, dtype=torch.uint8),
                    **tables()), dict(num_heads=4, kv_heads=2)
    return dict(logits=torch.zeros(2, 8), noise=torch.ones(2, 8), temperature=torch.ones(2),
                top_k=torch.ones(2, dtype=I32), top_p=torch.ones(2), min_p=torch.ones(2), tokens=torch.zeros(2, dtype=torch.int64),
                logprobs=torch.zeros(2)), {}


NAMES = ["paged_kv_quantize", "paged_kv_dequantize", "paged_attention_quantized", "sample"]


@pytest.mark.parametrize("name,which", [(n, w) for n in NAMES for w in arguments(n)[0]])
@pytest.mark.parametrize("place", [-1, 1])
def test_every_tensor_must_be_on_the_device(world, name, which, place):
    """Each tensor in turn on the host or on another GPU: refused before any launch."""
    ops, library, places = world
    tensors, other = arguments(name)
    places[tensors[which].data_ptr()] = place
    with pytest.raises(ValueError, match="one CUDA device"):
        getattr(ops, name)(**tensors, **other)
    assert not library.calls


@pytest.mark.parametrize("name", NAMES)
def test_tensors_on_one_device_are_taken(world, name):
    ops, library, _ = world
    tensors, other = arguments(name)
    getattr(ops, name)(**tensors, **other)
    assert library.calls == ["b200ep_" + name]


@pytest.mark.parametrize("name", NAMES[:3])
@pytest.mark.parametrize("shape", [(4, 2), (1, 4), (4, 1, 2)])
def test_a_block_table_of_other_sequences_is_refused(world, name, shape):
    """A pool's table with more rows than there are sequences: its rows would be read as halves of others."""
    ops, library, _ = world
    tensors, other = arguments(name)
    tensors["block_table"] = torch.zeros(shape, dtype=I32)
    with pytest.raises(ValueError, match="block_table"):
        getattr(ops, name)(**tensors, **other)
    assert not library.calls


def test_a_workspace_that_is_smaller_than_its_size_says_is_refused(world):
    ops, library, _ = world
    tensors, other = arguments("paged_attention_quantized")
    tensors["workspace"] = torch.zeros(1, dtype=torch.uint8).expand(1 << 20)
    with pytest.raises(ValueError, match="contiguous"):
        ops.paged_attention_quantized(**tensors, **other)
    assert not library.calls


@pytest.mark.parametrize("name", NAMES)
def test_the_launch_is_on_the_tensors_device(world, monkeypatch, name):
    """Tensors on a device that is not the current one: it is current while the entry point runs, and not after."""
    ops, library, places = world
    tensors, other = arguments(name)
    for x in tensors.values():
        places[x.data_ptr()] = 3
    now, seen = [0], []

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *a):
            now[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_current_device", lambda: now[0])
    setattr(library, "b200ep_" + name, lambda *a: seen.append(now[0]) or 0)
    getattr(ops, name)(**tensors, **other)
    assert seen == [3] and now == [0]
