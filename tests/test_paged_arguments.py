"""What the paged cache's wrappers refuse, and how they are imported, without a GPU."""
import importlib.util

import pytest
import torch

from paged_cases import normal

from moss_tts._runtime import kernels as K, native


def test_the_module_loads_and_finds_the_stream_without_the_private_name(monkeypatch):
    """``torch._C._cuda_getCurrentRawStream`` is not a public name: without it the public call answers."""
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    spec = importlib.util.spec_from_file_location("moss_tts._runtime.kernels_again", K.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)

    class Stream:
        cuda_stream = 1234

    asked = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: asked.append(device) or Stream())
    assert module._raw_stream(3) == 1234 and asked == [3]


BF = torch.bfloat16


def test_outputs_in_the_memory_of_inputs_are_named():
    """``_apart`` goes by addresses and strides, so host tensors show it."""
    memory = torch.zeros(64, 4, 64, dtype=BF)
    q = normal(400, 2, 4, 64)
    for other in (memory[10:20], memory[10:20, :2], memory[10:20].transpose(0, 1), memory.view(4, 16, 4, 64)[:, 3:9].transpose(1, 2)):
        for out in (memory[10:12], memory[11:13]):
            with pytest.raises(ValueError, match="out must not lie in the memory of k"):
                K._apart({"out": out}, {"the queries": q, "k": other, "cu_seqlens_k": None})
    with pytest.raises(ValueError, match="the queries"):
        K._apart({"out": q}, {"the queries": q})
    K._apart({"out": memory[20:22]}, {"the queries": memory[10:20], "k": memory[22:30]})
    K._apart({"out": memory[8:10]}, {"the queries": memory[10:20, :2], "k": memory[8:8]})  # nothing lies there
    pool = torch.zeros(3, 2, 2, 16, 64, dtype=BF)  # keys and values of a page side by side
    K._apart({"out": q, "k_pages": pool[:, 0], "v_pages": pool[:, 1]}, {"qkv": memory})
    with pytest.raises(ValueError, match="v_pages must not lie in the memory of qkv"):
        K._apart({"out": q, "k_pages": pool[0], "v_pages": pool[1]}, {"qkv": pool[1, 0]})
    with pytest.raises(ValueError, match="out must not lie in the memory of k_pages"):
        K._apart({"out": pool[0, 0, 0, :2], "k_pages": pool[0], "v_pages": pool[1]}, {"qkv": memory})


def test_the_write_refuses_outputs_in_the_memory_of_inputs():
    """The entry point itself, with addresses that nothing reads: 1 where it refuses, else what a machine without
    a GPU answers to a launch."""
    lib, far = native.library(), 1 << 30
    if torch.cuda.is_available():
        pytest.skip("the calls that are not refused would run")

    def call(qkv=far, q_norm=2 * far, cos=3 * far, table=4 * far, lens=5 * far, cu=6 * far, k=7 * far, v=8 * far, out=9 * far):
        kv = native.PAGED_KV.pack(k, v, table, lens, 4096, 1024, 64, 4096, 1024, 64, 4, 3, 2, 16, 64, 4, 2, 0)
        return lib.mt_qk_rope_paged(qkv, q_norm, q_norm + 128, cos, cos + 8192, 64, 0, kv, cu, 2, 4, 512, out, 1e-6, None, 0, None)

    page_bytes, row_bytes = 2 * (2 * 4096 + 1024 + 15 * 64 + 64), 2 * 4 * 64 * 2
    assert call() != 1
    for where, size in (("qkv", 2048), ("q_norm", 256), ("cos", 16384), ("table", 32), ("lens", 8), ("cu", 12)):
        for out, length in (("out", row_bytes), ("k", page_bytes), ("v", page_bytes)):
            at = 20 * far
            assert call(**{out: at, where: at + length - 16}) == 1, (where, out)
            assert call(**{out: at, where: at + length}) != 1, (where, out)
            if size > 32:
                assert call(**{out: at + size - 16, where: at}) == 1, (where, out)
            assert call(**{out: at + -(-size // 16) * 16, where: at}) != 1, (where, out)
    for page in ("k", "v"):
        assert call(out=20 * far, **{page: 20 * far + row_bytes - 16}) == 1
        assert call(out=20 * far, **{page: 20 * far + row_bytes}) != 1
    assert call(k=20 * far, v=20 * far + 2048) != 1  # keys and values side by side
