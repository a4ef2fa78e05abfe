"""Refusals of the window attention, filtered sampling and cache page calls, on the host and without a GPU."""
import pytest
import torch


def test_tensors_have_to_be_on_a_gpu():
    from llm_from_scratch_b200 import ops
    q, k = torch.zeros(2, 4, 64), torch.zeros(3, 16, 2, 64)
    bt, ids = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.window_decode(q, k, k, bt, torch.ones(2, dtype=torch.int64), 1.0, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.window_attention(q, k, k, bt, torch.arange(3).int(), torch.arange(3).int(), 1, 1.0, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_filtered(torch.zeros(2, 9), torch.zeros(2), torch.ones(2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagePools([k])
    with pytest.raises(ValueError, match="a pool"):
        ops.PagePools([])


class _Tensor(torch.Tensor):
    """A host tensor that says it is on device 0: the checks of the wrappers run before anything is launched."""
    is_cuda = True

    def get_device(self):
        return 0

    @property
    def device(self):
        return torch.device("cuda", 0)


@pytest.fixture
def ops(monkeypatch):
    from llm_from_scratch_b200 import ops

    def launch(*_):
        raise AssertionError("a call that should be refused was launched")

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(ops, "_stream", launch)
    monkeypatch.setattr(ops, "status_word", launch)
    return ops


def gpu(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Tensor)


def test_window_attention_refuses(ops, monkeypatch):
    i32, i64 = torch.int32, torch.int64
    good = dict(q=gpu(5, 4, 64), k_cache=gpu(3, 16, 2, 64), v_cache=gpu(3, 16, 2, 64), block_tables=gpu(2, 3, dtype=i32),
                cu_seqlens_q=gpu(3, dtype=i32), cu_seqlens_k=gpu(3, dtype=i32), max_seqlen_q=3, scale=1.0, window=8, first=2,
                out=gpu(5, 4, 64))
    bad = [dict(window=0), dict(window=-1), dict(window=1 << 31), dict(first=-1), dict(first=1 << 31), dict(max_seqlen_q=-1),
           dict(q=gpu(5, 3, 64)), dict(q=gpu(5, 256)), dict(q=gpu(5, 4, 63)), dict(q=gpu(5, 4, 64, dtype=torch.bfloat16)), dict(q=gpu(5, 64, 4).transpose(1, 2)),
           dict(k_cache=gpu(3, 8, 2, 64)), dict(v_cache=gpu(3, 16, 2, 64, dtype=torch.bfloat16)), dict(k_cache=gpu(3, 16, 64, 2).transpose(2, 3)),
           dict(block_tables=gpu(2, 3, dtype=i64)), dict(block_tables=gpu(3, 3, dtype=i32)), dict(block_tables=gpu(2, 6, dtype=i32)[:, ::2]),
           dict(block_tables=gpu(2, 0, dtype=i32)), dict(cu_seqlens_q=gpu(3, dtype=i64)), dict(cu_seqlens_k=gpu(4, dtype=i32)),
           dict(cu_seqlens_q=gpu(0, dtype=i32), cu_seqlens_k=gpu(0, dtype=i32)), dict(out=gpu(5, 4, 32)), dict(out=gpu(5, 4, 64, dtype=torch.bfloat16)),
           dict(out=gpu(5, 64, 4).transpose(1, 2))]
    for change in bad:
        with pytest.raises(ValueError):
            ops.window_attention(**{**good, **change})
    with pytest.raises(AssertionError, match="launched"):            # the good call passes the checks
        ops.window_attention(**good)
    for dtype in (torch.float16, torch.float64):
        cast = {n: gpu(*good[n].shape, dtype=dtype) for n in ("q", "k_cache", "v_cache", "out")}
        with pytest.raises(TypeError):
            ops.window_attention(**{**good, **cast})
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        ops.window_attention(**good)


def test_window_decode_refuses(ops):
    good = dict(q=gpu(2, 4, 64), k_cache=gpu(3, 16, 2, 64), v_cache=gpu(3, 16, 2, 64), block_tables=gpu(2, 3, dtype=torch.int32),
                context_lens=gpu(2, dtype=torch.int64), scale=1.0, window=8, first=2,
                out=gpu(2, 4, 64))
    for change in (dict(window=0), dict(first=-1), dict(context_lens=gpu(2, dtype=torch.int32)), dict(context_lens=gpu(3, dtype=torch.int64)),
                   dict(q=gpu(2, 5, 64)), dict(q=gpu(2, 8, 64)[:, ::2]), dict(block_tables=gpu(1, 3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.window_decode(**{**good, **change})
    with pytest.raises(AssertionError, match="launched"):
        ops.window_decode(**good)


def test_sample_filtered_refuses(ops):
    good = dict(logits=gpu(4, 100), uniforms=gpu(4), temperatures=gpu(4), top_k=gpu(4, dtype=torch.int32), top_p=gpu(4), min_p=gpu(4),
                out=gpu(4, dtype=torch.int64))
    for change in (dict(logits=gpu(400)), dict(logits=gpu(4, 0)), dict(logits=gpu(100, 4).t()), dict(logits=gpu(1, 100).expand(4, 100)),
                   dict(uniforms=gpu(3)), dict(temperatures=gpu(4, dtype=torch.float64)), dict(top_k=gpu(4, dtype=torch.int64)),
                   dict(top_p=gpu(8)[::2]), dict(min_p=gpu(5)), dict(out=gpu(4, dtype=torch.int32)), dict(out=gpu(5, dtype=torch.int64))):
        with pytest.raises(ValueError):
            ops.sample_filtered(**{**good, **change})
    with pytest.raises(TypeError):
        ops.sample_filtered(**{**good, "logits": gpu(4, 100, dtype=torch.float16)})
    with pytest.raises(AssertionError, match="launched"):
        ops.sample_filtered(**good)


def test_argument_errors_of_the_library():
    """Checks behind the wrappers, which come before any CUDA call."""
    from llm_from_scratch_b200._lib import lib
    x = 4096                                                          # an address that is never used
    att = lambda **c: lib.b200_window_attention(*{**dict(
        q=x, qs=256, k=x, v=x, out=x, total=4, cuq=x, cuk=x, n=1, longest=4, Hq=4, Hkv=2, D=64, Dv=64, scale=1.0, bt=x, stride=2, width=2, bs=16, nb=3,
        window=8, first=0, dtype=0, status=None, stream=None), **c}.values())
    assert att(Hq=3) == att(window=0) == att(first=-1) == att(bs=0) == att(width=0) == att(q=None) == att(cuq=None) == att(total=-1) == -1
    assert att(dtype=5) == att(D=1025) == att(Dv=2000) == -3
    assert att(n=0) == att(total=0) == att(longest=0) == 0
    dec = lambda **c: lib.b200_window_decode(*{**dict(q=x, k=x, v=x, out=x, bt=x, stride=2, width=2, lens=x, batch=1, Hq=4, Hkv=2, D=64, Dv=64, bs=16, nb=3,
                                                      scale=1.0, window=8, first=0, dtype=0, status=None, stream=None), **c}.values())
    assert dec(Hkv=3) == dec(window=-2) == dec(lens=None) == dec(bt=None) == -1 and dec(dtype=2) == -3 and dec(batch=0) == 0
    smp = lambda **c: lib.b200_sample_filtered(*{**dict(logits=x, stride=9, rows=1, vocab=9, u=x, t=x, k=None, p=None, m=None, out=x, ws=None, nbytes=0, dtype=0, stream=None), **c}.values())
    assert smp(vocab=0) == smp(stride=8) == smp(u=None) == smp(t=None) == smp(out=None) == -1
    assert smp(dtype=3) == -3 and smp(rows=0) == 0 and smp(vocab=(1 << 24) + 1, stride=1 << 25) == smp(rows=1 << 31) == -8
    need = lib.b200_sample_filtered_workspace_bytes(300, 131072)
    assert need > 0 and lib.b200_sample_filtered_workspace_bytes(1, 100) == lib.b200_sample_filtered_workspace_bytes(0, 131072) == 0
    assert smp(rows=300, vocab=131072, stride=131072) == smp(rows=300, vocab=131072, stride=131072, ws=x, nbytes=need - 1) == -5
    cpy = lambda **c: lib.b200_copy_pages(*{**dict(pools=x, sizes=x, largest=64, n=1, pages=5, source=x, target=x, pairs=2, ws=None, nbytes=0, status=None, stream=None), **c}.values())
    assert cpy(pairs=-1) == cpy(source=None) == cpy(pools=None) == -1 and cpy(pairs=0) == cpy(n=0) == 0
    assert lib.b200_copy_pages_workspace_bytes(1024, 700) == 0 and lib.b200_copy_pages_workspace_bytes(1025, 700) == 2800
    assert cpy(pairs=1025) == cpy(pairs=1025, ws=x, nbytes=19) == -5 and cpy(pairs=0x7fffffff) == cpy(pages=1 << 31) == -8
    cmp_ = lambda **c: lib.b200_compact_pages(*{**dict(pools=x, sizes=x, largest=64, n=1, pages=5, bt=x, stride=2, rows=3, width=2, out=x, map=x, source=x, target=x, counts=x,
                                                       status=None, stream=None), **c}.values())
    assert cmp_(stride=1) == cmp_(bt=None) == cmp_(map=None) == cmp_(counts=None) == cmp_(rows=-1) == -1 and cmp_(pages=1 << 31) == -8


def test_page_ids_are_checked(ops):
    pools = object.__new__(ops.PagePools)
    pools.tensors, pools.num_pages = [gpu(4, 16, 2, 64)], 4
    ids = gpu(3, dtype=torch.int32)
    for a, b in ((gpu(3, dtype=torch.int64), ids), (ids, gpu(2, dtype=torch.int32)), (gpu(6, dtype=torch.int32)[::2], ids), (ids, gpu(3, 1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.copy_pages(pools, a, b)
    for t in (gpu(3, 2), gpu(6, dtype=torch.int32), gpu(3, 4, dtype=torch.int32)[:, ::2]):
        with pytest.raises(ValueError):
            ops.compact_pages(pools, t)


def test_pools_are_checked(ops):
    for pools in ([gpu(4, 8), gpu(5, 8)], [gpu(4, 8).t()], [gpu()]):
        with pytest.raises(ValueError):
            ops.PagePools(pools)
    one = gpu(8, 4)
    with pytest.raises(ValueError, match="overlap"):
        ops.PagePools([one[:4], one[2:6]])
