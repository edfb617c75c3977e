"""Host side of the kv_* calls and of residual_rms_norm, runnable without a GPU: sizes, refusals, native arguments, and the
test suite's own model of the 8-bit rounding."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from raftinfer_b200 import _call, _lib
from raftinfer_b200 import kernels as K
from kv_util import E4M3_VALUES, codes_for, scale_for

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = {"kv_attention_prefill": "rib200_kv_attention_prefill", "kv_paged_prefill": "rib200_kv_paged_prefill",
         "kv_batched_decode": "rib200_kv_batched_decode", "kv_paged_decode": "rib200_kv_paged_decode",
         "residual_rms_norm": "rib200_residual_rms_norm"}


def test_sizes():
    assert K.kv_cache_bytes(4, 256, K.KV_BF16) == 2 * 4 * 256 * 256 * 2
    assert K.kv_cache_bytes(4, 256, K.KV_E4M3) == 2 * 4 * 16 * 4112
    assert K.kv_cache_bytes(3, 17, K.KV_E4M3) == 2 * 3 * 2 * 4112
    shape = K.Qwen35AttentionShape(100, 16, 4, 256, 5000, 3000)
    rows = lambda n: 2 * 4 * 256 * 2 * n
    workspace = lambda window, sinks, kind=K.KV_E4M3, paged=False: K.kv_prefill_workspace_bytes(shape, window, sinks, kind, paged)
    assert workspace(0, 0) == rows(3100) and workspace(0, 9) == rows(3100)
    assert workspace(1000, 0) == rows(1099) and workspace(1000, 5) == rows(1104) and workspace(1, 0) == rows(100)
    # sinks up to 2099 (the last query's window has passed them) and tokens from 2001 on: 2100 + 1099 - 99 that are both
    assert workspace(1000, 2200) == rows(3100)
    assert workspace(1000, 5, K.KV_BF16) == 0 and workspace(1000, 5, K.KV_BF16, True) == rows(1104)
    assert K.kv_decode_workspace_bytes() > 0
    for call, code in ((lambda: K.kv_cache_bytes(0, 1, K.KV_BF16), K.INVALID_ARGUMENT),
                       (lambda: K.kv_cache_bytes(1, 0, K.KV_BF16), K.INVALID_ARGUMENT),
                       (lambda: K.kv_cache_bytes(1, 1, K.KV_F32), K.UNSUPPORTED),
                       (lambda: K.kv_cache_bytes(1, 1, 7), K.INVALID_ARGUMENT),
                       (lambda: K.kv_cache_bytes(2 ** 40, 2 ** 40, K.KV_E4M3), K.INVALID_ARGUMENT)):
        with pytest.raises(K.Qwen35PrimitiveError) as refusal:
            call()
        assert refusal.value.code == code


def refused(call, good, changes):
    for change, code, text in changes:
        with pytest.raises(K.Qwen35PrimitiveError, match=text) as refusal:
            call(**{**good, **change})
        assert refusal.value.code == code, change


POINTERS = [({name: None}, K.INVALID_ARGUMENT, "pointer is null") for name in ("query", "key", "value", "gate", "output")]
POINTERS += [({name: 24}, K.INVALID_ARGUMENT, f"{name} is not 16-byte aligned")
             for name in ("query", "key", "value", "gate", "output")]
ACTIVATIONS = POINTERS + [({"stream": None}, K.INVALID_ARGUMENT, "stream is null"),
                          ({"activation_dtype": 9}, K.INVALID_ARGUMENT, "unknown activation dtype"),
                          ({"activation_dtype": K.DTYPE_F16}, K.UNSUPPORTED, "FP32 or BF16"),
                          ({"cache_dtype": 9}, K.INVALID_ARGUMENT, "unknown KV cache dtype"),
                          ({"cache_dtype": K.KV_F32}, K.UNSUPPORTED, "BF16 or E4M3")]
SHAPE = dict(tokens=100, query_heads=16, kv_heads=4, head_dim=256, max_context_tokens=512, past_tokens=300)
SHAPES = [(dict(shape=K.Qwen35AttentionShape(**{**SHAPE, **change})), code, text) for change, code, text in
          [({"tokens": 0}, K.INVALID_ARGUMENT, "tokens must be positive"),
           ({"query_heads": 0}, K.INVALID_ARGUMENT, "head counts must be positive"),
           ({"kv_heads": 0}, K.INVALID_ARGUMENT, "head counts must be positive"),
           ({"query_heads": 15}, K.INVALID_ARGUMENT, "multiple of kv_heads"),
           ({"head_dim": 128}, K.UNSUPPORTED, "head_dim 256"),
           ({"past_tokens": 413}, K.INVALID_ARGUMENT, "exceeds the cache capacity"),
           ({"past_tokens": 2 ** 64 - 50}, K.INVALID_ARGUMENT, "exceeds the cache capacity"),
           ({"query_heads": 2048}, K.UNSUPPORTED, "1024 query heads"),
           ({"query_heads": 1024, "kv_heads": 512}, K.UNSUPPORTED, "256 KV heads"),
           ({"past_tokens": 2 ** 23, "max_context_tokens": 2 ** 24}, K.UNSUPPORTED, "2\\^23")]]


def test_prefill_refuses():
    good = dict(query=16, key=16, value=16, gate=16, output=16, kv_cache=16, kv_cache_bytes=1 << 40, workspace=16,
                workspace_bytes=1 << 40, shape=K.Qwen35AttentionShape(**SHAPE), window_tokens=64, sink_tokens=4,
                activation_dtype=K.DTYPE_BF16, cache_dtype=K.KV_E4M3, stream=16)
    need = K.kv_prefill_workspace_bytes(good["shape"], 64, 4, K.KV_E4M3)
    refused(K.kv_attention_prefill, good, ACTIVATIONS + SHAPES + [
        ({"kv_cache": None}, K.INVALID_ARGUMENT, "KV cache pointer is null"),
        ({"kv_cache": 8}, K.INVALID_ARGUMENT, "KV cache is not 16-byte aligned"),
        ({"kv_cache_bytes": K.kv_cache_bytes(4, 512, K.KV_E4M3) - 1}, K.INVALID_ARGUMENT, "KV cache is too small"),
        ({"workspace": None}, K.INVALID_ARGUMENT, "workspace is null"),
        ({"workspace": 40}, K.INVALID_ARGUMENT, "workspace is not 16-byte aligned"),
        ({"workspace_bytes": need - 1}, K.INVALID_ARGUMENT, "workspace is too small")])


def test_paged_prefill_refuses():
    good = dict(query=16, key=16, value=16, gate=16, output=16, page_pool=16, pool_pages=9, block_table=16, max_blocks=2,
                workspace=16, workspace_bytes=1 << 40, shape=K.Qwen35AttentionShape(**SHAPE), window_tokens=0, sink_tokens=0,
                activation_dtype=K.DTYPE_BF16, cache_dtype=K.KV_BF16, stream=16)
    refused(K.kv_paged_prefill, good, ACTIVATIONS + SHAPES[:9] + [
        ({"page_pool": None}, K.INVALID_ARGUMENT, "page pool or the block table pointer is null"),
        ({"block_table": None}, K.INVALID_ARGUMENT, "page pool or the block table pointer is null"),
        ({"page_pool": 8}, K.INVALID_ARGUMENT, "page pool is not 16-byte aligned"),
        ({"pool_pages": 0}, K.INVALID_ARGUMENT, "pool_pages out of range"),
        ({"max_blocks": 0}, K.INVALID_ARGUMENT, "blocks per sequence out of range"),
        ({"max_blocks": 3}, K.INVALID_ARGUMENT, "256 \\* max_blocks"),
        ({"workspace": None}, K.INVALID_ARGUMENT, "workspace is null"),
        ({"workspace_bytes": 100}, K.INVALID_ARGUMENT, "workspace is too small")])


DECODES = [({"positions": None}, K.INVALID_ARGUMENT, "positions pointer is null"),
           ({"batch": 0}, K.INVALID_ARGUMENT, "batch must be in"), ({"batch": 65536}, K.INVALID_ARGUMENT, "batch must be in"),
           ({"query_heads": 0}, K.INVALID_ARGUMENT, "head counts must be positive"),
           ({"kv_heads": 0}, K.INVALID_ARGUMENT, "head counts must be positive"),
           ({"kv_heads": 3}, K.INVALID_ARGUMENT, "multiple of kv_heads"),
           ({"kv_heads": 2}, K.UNSUPPORTED, "1 to 4 query heads"),
           ({"query_heads": 257, "kv_heads": 257}, K.UNSUPPORTED, "256 KV heads"),
           ({"workspace": None}, K.INVALID_ARGUMENT, "workspace is null"),
           ({"workspace": 8}, K.INVALID_ARGUMENT, "workspace is not 16-byte aligned"),
           ({"workspace_bytes": 100}, K.INVALID_ARGUMENT, "workspace is too small")]


def test_decode_refuses():
    common = dict(query=16, key=16, value=16, gate=16, output=16, positions=16, batch=3, query_heads=16, kv_heads=4,
                  window_tokens=0, sink_tokens=0, activation_dtype=K.DTYPE_F32, cache_dtype=K.KV_E4M3, workspace=16,
                  workspace_bytes=1 << 40, stream=16)
    refused(K.kv_batched_decode, dict(common, kv_caches=16, max_context_tokens=16), ACTIVATIONS + DECODES + [
        ({"kv_caches": None}, K.INVALID_ARGUMENT, "cache or capacity array is null"),
        ({"max_context_tokens": None}, K.INVALID_ARGUMENT, "cache or capacity array is null")])
    refused(K.kv_paged_decode, dict(common, page_pool=16, pool_pages=5, block_tables=16, max_blocks_per_sequence=3),
            ACTIVATIONS + DECODES + [
        ({"page_pool": None}, K.INVALID_ARGUMENT, "page pool or the block table pointer is null"),
        ({"block_tables": None}, K.INVALID_ARGUMENT, "page pool or the block table pointer is null"),
        ({"page_pool": 8}, K.INVALID_ARGUMENT, "page pool is not 16-byte aligned"),
        ({"pool_pages": 2 ** 40}, K.INVALID_ARGUMENT, "pool_pages out of range"),
        ({"max_blocks_per_sequence": 2 ** 23}, K.INVALID_ARGUMENT, "blocks per sequence out of range")])


def test_residual_norm_refuses():
    good = dict(input=16, residual=16, weight=16, output=16, scales=16, residual_out=16, rows=3, columns=512,
                group_columns=128, epsilon=1e-6, dtype=K.DTYPE_BF16, weight_dtype=K.DTYPE_F32, output_dtype=K.DTYPE_E4M3,
                stream=16)
    plain = dict(scales=None, group_columns=0, output_dtype=K.DTYPE_BF16)
    refused(K.residual_rms_norm, good, [
        ({"input": None}, K.INVALID_ARGUMENT, "pointer is null"), ({"weight": None}, K.INVALID_ARGUMENT, "pointer is null"),
        ({"output": None}, K.INVALID_ARGUMENT, "pointer is null"), ({"stream": None}, K.INVALID_ARGUMENT, "stream is null"),
        ({"scales": None}, K.INVALID_ARGUMENT, "scales pointer is null"),
        ({"scales": 18}, K.INVALID_ARGUMENT, "4-byte aligned"),
        ({"rows": 0}, K.INVALID_ARGUMENT, "must be positive"), ({"columns": 0}, K.INVALID_ARGUMENT, "must be positive"),
        ({"rows": 2 ** 31}, K.INVALID_ARGUMENT, "too many rows"),
        ({"columns": 510}, K.UNSUPPORTED, "multiple of 8"), ({"columns": 16392}, K.UNSUPPORTED, "up to 16384"),
        ({"columns": 520}, K.INVALID_ARGUMENT, "multiple of group_columns"),
        ({"group_columns": 64}, K.UNSUPPORTED, "32 or 128"),
        ({"epsilon": -1.0}, K.INVALID_ARGUMENT, "epsilon"), ({"epsilon": float("nan")}, K.INVALID_ARGUMENT, "epsilon"),
        ({"dtype": 0}, K.INVALID_ARGUMENT, "unknown dtype"), ({"dtype": 4}, K.INVALID_ARGUMENT, "unknown dtype"),
        ({"weight_dtype": 7}, K.INVALID_ARGUMENT, "unknown weight dtype"),
        ({"weight_dtype": K.DTYPE_F16}, K.UNSUPPORTED, "weights are FP32 or BF16"),
        ({"output_dtype": 5}, K.INVALID_ARGUMENT, "unknown output dtype"),
        ({**plain, "output_dtype": K.DTYPE_F32}, K.UNSUPPORTED, "input's dtype or E4M3"),
        ({**plain, "scales": 16}, K.INVALID_ARGUMENT, "scales belong"),
        ({**plain, "group_columns": 128}, K.INVALID_ARGUMENT, "scales belong"),
        *[({name: 24}, K.INVALID_ARGUMENT, f"{name} is not 16-byte aligned")
          for name in ("input", "residual", "weight", "output", "residual_out")]])


# ---- the native functions ----
class Tensor:
    def __init__(self, address):
        self.address = address

    def data_ptr(self):
        return self.address


class Stream:
    cuda_stream = 0x5EED_0000_0001


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    """call(name, arguments, native) -> the bytes that arrive, or the exception's type."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    library = str(tmp_path_factory.mktemp("stub") / "librecording.so")
    subprocess.run([cxx, "-std=c++17", "-O1", "-fPIC", "-shared",
                    os.path.join(ROOT, "tests", "cpp", "kv_recording_stub.cpp"), "-o", library], check=True)
    stub = ctypes.CDLL(library)
    stub.stub_address.argtypes, stub.stub_address.restype = [ctypes.c_char_p], ctypes.c_void_p
    stub.stub_record.argtypes, stub.stub_record.restype = [ctypes.c_void_p, ctypes.c_size_t], ctypes.c_size_t
    buffer = ctypes.create_string_buffer(4096)

    def call(name, arguments, native):
        entry = NAMES[name]
        try:
            if native:
                getattr(_call, name)(*arguments)
            else:
                function = ctypes.CFUNCTYPE(_lib.Status, *_lib.PROTOTYPES[entry])(stub.stub_address(entry.encode()))
                assert function(*K._ctypes_arguments(entry, arguments)).code == 0
        except Exception as error:  # noqa: BLE001 - the type is what is compared
            stub.stub_record(buffer, len(buffer))
            return type(error)
        arrived = stub.stub_record(buffer, len(buffer))
        return buffer.raw[:arrived]

    _call.bind_more(lambda name: stub.stub_address(name.encode()))
    yield call
    _call.bind_more(lambda name: ctypes.cast(getattr(_lib.lib, name), ctypes.c_void_p).value)


@pytest.mark.parametrize("name", list(NAMES))
def test_every_argument_arrives_as_through_ctypes(name, recorder):
    count = iter(range(1, 1000))
    make = {_lib.AttentionShape: lambda: K.Qwen35AttentionShape(*[(1 << 40) + next(count) for _ in range(6)]),
            _lib.vp: lambda: Tensor((1 << 44) + 16 * next(count)), _lib.sz: lambda: (1 << 40) + next(count),
            ctypes.c_int32: lambda: -next(count), ctypes.c_uint8: lambda: next(count), ctypes.c_float: lambda: 0.5 + next(count)}
    types = _lib.PROTOTYPES[NAMES[name]]
    arguments = [make[getattr(t, "_type_", None) if hasattr(t, "_type_") and not isinstance(t._type_, str) else t]()
                 for t in types]
    arguments[-1] = Stream()
    native = recorder(name, arguments, True)
    assert isinstance(native, bytes) and native and native == recorder(name, arguments, False)
    for i in range(len(arguments)):
        for other in [None, 0, 7, -1, 2 ** 31, 2 ** 64 - 1]:
            changed = arguments[:i] + [other] + arguments[i + 1:]
            first = recorder(name, changed, True)
            if isinstance(first, bytes):
                assert first == recorder(name, changed, False), (i, other)
    for wrong in (len(types) - 1, len(types) + 1):
        with pytest.raises(TypeError):
            getattr(_call, name)(*[None] * wrong)


# ---- the model of the rounding that the GPU tests compare with ----
def test_the_model_rounds_as_torch_does():
    x = torch.cat([torch.randn(4000, generator=torch.Generator().manual_seed(1)) * 2.0 ** k for k in range(-12, 8)])
    x = x.clamp(-448, 448)
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes_for(x.double().numpy()), want)
    halves = (E4M3_VALUES[:126] + E4M3_VALUES[1:127]) / 2  # exactly between two codes: the even one
    assert (codes_for(halves) % 2 == 0).all()
    assert codes_for([1e9, -np.inf, np.nan, 0.0]).tolist() == [0x7E, 0xFE, 0x7F, 0]


def test_the_model_of_the_scale():
    for e in (-90, -3, 0, 5, 100):
        assert scale_for(448.0 * 2.0 ** e) == 2.0 ** e
        assert scale_for(np.nextafter(448.0 * 2.0 ** e, np.inf)) == 2.0 ** (e + 1)
        assert scale_for(225.0 * 2.0 ** e) == 2.0 ** e and scale_for(224.0 * 2.0 ** e) == 2.0 ** (e - 1)
    assert scale_for(0.0) == 2.0 ** -100 == scale_for(2.0 ** -140) and scale_for(2.0 ** 127.9) == 2.0 ** 119


@pytest.mark.parametrize("cache_dtype", [K.KV_BF16, K.KV_E4M3])
def test_a_prompt_workspace_holds_each_visible_row_once(cache_dtype):
    """Sinks that lie in the first token's window, next to it, and in front of it: never more rows than the call sees."""
    row = 2 * 4 * 256 * 2
    for tokens, past, window, sinks in ((988, 0, 83, 163), (988, 0, 83, 905), (988, 0, 83, 2000), (100, 500, 200, 301),
                                        (100, 500, 200, 300), (100, 500, 200, 302), (100, 500, 200, 0), (100, 500, 200, 350),
                                        (100, 500, 0, 0), (100, 500, 1000, 7), (1, 500, 1, 500), (1, 0, 1, 1)):
        first_low = max(0, past + 1 - window) if window else 0
        last_low = max(0, past + tokens - window) if window else 0
        seen = set(range(first_low, past + tokens)) | set(range(min(sinks, last_low)))
        shape = K.Qwen35AttentionShape(tokens, 16, 4, 256, 4096, past)
        assert K.kv_prefill_workspace_bytes(shape, window, sinks, cache_dtype, True) == len(seen) * row, (tokens, past, window, sinks)
