"""Tensors of several GPUs in one call (no GPU needed: what the calls ask of a tensor is stood in for)."""

from types import SimpleNamespace

import pytest
import torch

from h3b import cache, streaming


def _on(gpu, shape=(4, 2, 128), dtype=torch.bfloat16):
    x = torch.zeros(shape, dtype=dtype)
    return SimpleNamespace(get_device=lambda: gpu, is_cuda=gpu >= 0, shape=x.shape, ndim=x.ndim, dtype=dtype,
                           stride=x.stride, data_ptr=lambda: 16, is_contiguous=lambda: True, numel=x.numel,
                           element_size=x.element_size, new_empty=x.new_empty)


def _cache_on(**other):
    ints = dict(dtype=torch.int32)
    parts = dict(k=_on(0, (1, 4, 2, 16, 128)), v=_on(0, (1, 4, 2, 16, 128)), table=_on(0, (3, 8), **ints),
                 lens=_on(0, (3,), **ints), refs=_on(0, (4,), **ints), status=_on(0, (1,), **ints))
    return cache.PagedKVCache(**(parts | other))


def test_a_call_gets_the_stream_of_its_tensors_gpu(monkeypatch):
    monkeypatch.setattr(cache, "_current_gpu", lambda: 1)
    monkeypatch.setattr(cache, "_raw_stream", lambda gpu: 100 + gpu)
    assert cache._stream(1) == 101
    with pytest.raises(RuntimeError, match="on cuda:0, the current device is cuda:1"):
        cache._stream(0)


@pytest.mark.parametrize("gpu", [1, -1])  # -1: not a GPU's
def test_parts_of_a_cache_on_another_gpu_are_refused(gpu):
    assert _cache_on()._gpu == 0
    for part in ("v", "table", "lens", "refs", "status"):
        kind = getattr(_cache_on(), part)
        with pytest.raises(ValueError, match="one GPU"):
            _cache_on(**{part: _on(gpu, kind.shape, kind.dtype)})
    e4m3 = {x: _on(0, (1, 4, 2, 16, 128), torch.float8_e4m3fn) for x in "kv"}
    scale = _on(0, (1, 2), torch.float32)
    _cache_on(**e4m3, k_scale=scale, v_scale=scale)
    for part in ("k_scale", "v_scale"):
        with pytest.raises(ValueError, match="on its GPU"):
            _cache_on(**(e4m3 | dict(k_scale=scale, v_scale=scale) | {part: _on(gpu, (1, 2), torch.float32)}))


@pytest.mark.parametrize("gpu", [1, -1])
def test_tensors_of_another_gpu_are_refused(gpu):
    c, x, ints = _cache_on(), _on(0), dict(shape=(4,), dtype=torch.int32)
    other, ids, other_ids = _on(gpu), _on(0, **ints), _on(gpu, **ints)
    for call in (lambda: streaming.window_attention(x, other, x), lambda: streaming.window_attention(x, x, other),
                 lambda: streaming.decode_attention(other, c), lambda: streaming.paged_window_attention(other, c),
                 lambda: c.append(ids, other, x), lambda: c.write(ids, x, other)):
        with pytest.raises((ValueError, RuntimeError), match="GPU|CUDA"):
            call()
    for call in (lambda: streaming.decode_attention(x, c, other_ids), lambda: c.append(other_ids, x, x),
                 lambda: streaming.paged_window_attention(x, c, query_starts=other_ids), lambda: c.extend(other_ids),
                 lambda: streaming.window_attention(x, x, x, query_starts=other_ids, key_starts=ids),
                 lambda: streaming.window_attention(x, x, x, query_starts=ids, key_starts=other_ids),
                 lambda: c.write(ids, x, x, other_ids), lambda: c.fork(ids, other_ids), lambda: c.fork(other_ids, ids),
                 lambda: c.truncate(ids, other_ids), lambda: c.free(other_ids), lambda: c.copy_pages(ids, other_ids)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="GPU"):
        streaming._output(other, x)
    with pytest.raises(ValueError, match="GPU"):
        streaming._workspace(_on(gpu, (64,), torch.uint8), 64, x)
