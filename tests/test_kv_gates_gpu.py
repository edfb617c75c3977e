"""Gates of any size in the kv_* calls: very small ones keep their relative precision, and a not-a-number stays one."""
import math

import numpy as np
import pytest
import torch

from raftinfer_b200 import kernels as K
from kv_util import D, HALF_STEP, Cache, activation, attention, normal, to_device

pytestmark = pytest.mark.gpu

GATES = [0.0, -39.0, -40.0, -41.0, -60.0, -86.0, 60.0, math.inf, -math.inf, -100.0, -3.0e38, math.nan, 3.0e38, -200.0]


def check(got, out, size, gate, weights, dtype):
    """`weights`: what the call's weights and logits may be off by, of `size`.  Gates under -87 may count as minus infinity: 2^-125 is
    more than their sigmoid."""
    got, gate = got.double(), gate.cuda()
    assert torch.equal(torch.isnan(got), torch.isnan(gate))
    rest = ~torch.isnan(gate)
    magnitude = size / torch.sigmoid(gate.double()).clamp_min(2.0 ** -1000)
    limit = size * weights + out.abs() * HALF_STEP[dtype] + torch.where(gate < -87.0, magnitude.clamp(0, 100.0) * 2.0 ** -125, 0.0)
    limit = torch.where(torch.isinf(gate) & (gate < 0), torch.zeros_like(limit), limit)
    off = (got - out).abs()
    assert (off[rest] <= limit[rest] + 2.0 ** -133).all()


@pytest.mark.parametrize("kind", [K.KV_BF16, K.KV_E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("dtype", [K.DTYPE_BF16, K.DTYPE_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("tokens,past,window", [(700, 0, 0), (700, 0, 300), (128, 1100, 0), (200, 1500, 0), (100, 4000, 0),
                                                (33, 0, 0)])
def test_prompts(kind, dtype, tokens, past, window):
    """Whole and split items, tiles of two boxes of rows and less."""
    heads, kv_heads = 16, 4
    query, q = activation(normal(1, tokens, heads, D), dtype)
    gate = normal(2, tokens, heads, D)
    gate.view(-1)[::37] = torch.tensor(GATES).repeat(gate.numel() // 37 // len(GATES) + 1)[:len(gate.view(-1)[::37])]
    gate, g = activation(gate, dtype)
    key, k = activation(normal(3, tokens, kv_heads, D), dtype)
    value, v = activation(normal(4, tokens, kv_heads, D), dtype)
    model = Cache(kind, kv_heads, past + tokens)
    if past:
        model.store(0, normal(5, 2, kv_heads, past, D).numpy())
    cache = to_device(model.bytes)
    shape = K.Qwen35AttentionShape(tokens, heads, kv_heads, D, past + tokens, past)
    need = K.kv_prefill_workspace_bytes(shape, window, 0, kind)
    workspace = torch.empty(need, device="cuda", dtype=torch.uint8) if need else None
    output = torch.empty_like(query)
    K.kv_attention_prefill(query, key, value, gate, output, cache, cache.numel() * cache.element_size(), workspace, need, shape,
                           window, 0, dtype, kind, torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    model.store(past, np.stack([k.permute(1, 0, 2).numpy(), v.permute(1, 0, 2).numpy()]))
    out, size, spread, total = attention(model, q, g, past, window, 0)
    # BF16 weights, 2^-14 for exponentials and the gate, and a logit's error twice, as in the tests of ordinary gates
    logit = 2.0 ** -16 + (2.0 ** -8 if dtype == K.DTYPE_F32 else 0.0)
    check(output, out, size, g, 2.0 ** -8 + 2.0 ** -14 + 2 * logit * spread, query.dtype)


@pytest.mark.parametrize("kind", [K.KV_BF16, K.KV_E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("dtype", [K.DTYPE_BF16, K.DTYPE_F32], ids=["bf16", "f32"])
def test_single_tokens(kind, dtype):
    from test_kv_decode_gpu import PARTS, SMALLEST, Batch

    b = Batch(kind, [300, 5, 1700], dtype, 9)
    b.g.view(-1)[::37] = torch.tensor(GATES).repeat(b.g.numel() // 37 // len(GATES) + 1)[:len(b.g.view(-1)[::37])]
    b.gate, b.g = activation(b.g, dtype)
    b.run()
    torch.cuda.synchronize()
    for i, length in enumerate(b.lengths):
        out, size, spread, total = attention(b.after[i], b.q[i:i + 1], b.g[i:i + 1], length - 1, 0, 0)
        weights = 4 * PARTS * spread + 4 * PARTS + SMALLEST * total / size.clamp_min(1e-300)
        check(b.output[i:i + 1], out, size, b.g[i:i + 1], weights, b.output.dtype)
