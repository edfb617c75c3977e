"""Prompts over BF16 and 8-bit caches, whole and windowed, against a plain 64-bit model."""
import numpy as np
import pytest
import torch

from raftinfer_b200 import kernels as K
from kv_util import D, HALF_STEP, PAGE, Cache, activation, attention, from_device, normal, to_device, visible

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", [K.KV_BF16, K.KV_E4M3], ids=["bf16", "e4m3"])


def tolerance(out, size, spread, dtype, f32_queries):
    """Weights are rounded to BF16 (half a step, 2^-8), FP32 queries too, and sums of 256 products in 32 bits are within 2^-16
    of their sum |q k| / 16; a logit's error counts twice (numerator and denominator).  2^-14: exponentials and the gate."""
    logit = 2.0 ** -16 + (2.0 ** -8 if f32_queries else 0.0)
    return size * (2.0 ** -8 + 2.0 ** -14 + 2 * logit * spread) + out.abs() * HALF_STEP[dtype] + 1e-30


class Prompt:
    def __init__(self, kind, capacity, kv_heads=4, group=4, window=0, sinks=0, paged=False, dtype=K.DTYPE_BF16, seed=1):
        self.kind, self.kv_heads, self.group, self.window, self.sinks = kind, kv_heads, group, window, sinks
        self.paged, self.dtype, self.seed, self.past = paged, dtype, seed, 0
        self.capacity = -(-capacity // PAGE) * PAGE if paged else capacity
        self.model = Cache(kind, kv_heads, self.capacity)
        if paged:
            blocks = self.capacity // PAGE
            self.pool_pages = blocks + 3
            self.order = np.random.default_rng(seed).permutation(self.pool_pages)[:blocks]
            pool = np.full((self.pool_pages, *self.model.pages().shape[1:]), 0x7F if kind == K.KV_E4M3 else 0x7FC1,
                           dtype=self.model.bytes.dtype)
            self.want = pool.copy()
            self.cache = to_device(pool)
        else:
            self.cache = to_device(self.model.bytes)

    def fill(self, tokens):
        """A past that the call under test did not make; rows that its first token does not see are not-a-numbers."""
        if tokens:
            self.model.store(0, normal(self.seed + 900, 2, self.kv_heads, tokens, D).numpy())
            if self.window:
                seen = set(visible(tokens, self.window, self.sinks)) | set(range(self.sinks))
                self.model.poison([t for t in range(tokens) if t not in seen])
        if self.paged:
            pool = self.want.copy()
            pool[self.order] = self.model.pages()
            self.cache.copy_(to_device(pool))
        else:
            self.cache.copy_(to_device(self.model.bytes))
        self.past = tokens

    def table(self, tokens):
        entries = np.full(self.capacity // PAGE, 0xFFFFFFFF, dtype=np.uint32)
        seen = visible(self.past, self.window, self.sinks) + list(range(self.past, self.past + tokens))
        if self.window:
            seen += list(range(min(self.sinks, self.past + tokens)))
        for b in {t // PAGE for t in seen}:
            entries[b] = self.order[b]
        return torch.from_numpy(entries.view(np.int32)).cuda()

    def chunk(self, tokens, stream=None, check=True):
        heads = self.kv_heads * self.group
        seed = self.seed + 10 + self.past
        query, q = activation(normal(seed, tokens, heads, D), self.dtype)
        gate, g = activation(2.0 * normal(seed + 1, tokens, heads, D), self.dtype)
        key, k = activation(normal(seed + 2, tokens, self.kv_heads, D), self.dtype)
        value, v = activation(normal(seed + 3, tokens, self.kv_heads, D), self.dtype)
        self.output = torch.full((tokens + 1, heads, D), 7.0, device="cuda", dtype=query.dtype)
        shape = K.Qwen35AttentionShape(tokens, heads, self.kv_heads, D, self.capacity, self.past)
        need = K.kv_prefill_workspace_bytes(shape, self.window, self.sinks, self.kind, self.paged)
        assert (need == 0) == (self.kind == K.KV_BF16 and not self.paged)
        workspace = torch.full((need + 64,), 0xFF, device="cuda", dtype=torch.uint8) if need else None  # not-a-numbers
        stream = stream or torch.cuda.current_stream()
        rest = (workspace, need, shape, self.window, self.sinks, self.dtype, self.kind, stream)
        if self.paged:
            table = self.table(tokens)
            K.kv_paged_prefill(query, key, value, gate, self.output, self.cache, self.pool_pages, table, len(table), *rest)
        else:
            K.kv_attention_prefill(query, key, value, gate, self.output, self.cache,
                                   self.cache.numel() * self.cache.element_size(), *rest)
        self.held = (query, key, value, gate, workspace)
        rows = np.stack([k.permute(1, 0, 2).numpy(), v.permute(1, 0, 2).numpy()])
        self.model.store(self.past, rows)
        past, self.past = self.past, self.past + tokens
        if check:
            torch.cuda.synchronize()
            assert K.device_status(torch.cuda.current_stream()) == 0
            out, size, spread, total = attention(self.model, q, g, past, self.window, self.sinks)
            limit = tolerance(out, size, spread, query.dtype, self.dtype == K.DTYPE_F32)
            off = (self.output[:tokens].double() - out).abs()
            assert (off <= limit).all(), (tokens, past, float((off / limit).max()))
            rel = float((self.output[:tokens].double() - out).norm() / out.norm())
            assert rel <= (1e-2 if self.dtype == K.DTYPE_F32 else 4e-3), rel
            assert (self.output[tokens] == 7.0).all(), "a row behind the last token was written"
            if need:
                assert (workspace[need:] == 0xFF).all()
            self.check_cache()

    def check_cache(self):
        if self.paged:
            want = self.want.copy()
            want[self.order] = self.model.pages()
        else:
            want = self.model.bytes
        assert np.array_equal(from_device(self.cache, want), want)


@KINDS
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("tokens,past", [(1, 0), (2, 0), (16, 0), (17, 3), (1, 15), (1, 16), (1, 300), (100, 0), (128, 128),
                                         (129, 0), (255, 1), (200, 1500), (700, 77), (1024, 0), (17, 2688), (300, 3000)])
def test_whole_context(kind, paged, tokens, past):
    p = Prompt(kind, past + tokens + (0 if paged else 13), paged=paged)
    p.fill(past)
    p.chunk(tokens)


@KINDS
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("tokens,past,window,sinks", [
    (1, 0, 1, 0), (1, 700, 1, 0), (1, 700, 5, 2), (130, 0, 1, 1), (300, 0, 20, 4), (300, 500, 64, 0), (513, 0, 128, 128),
    (400, 1000, 129, 3), (257, 130, 127, 200), (200, 2000, 1000, 17), (640, 64, 256, 500), (1000, 0, 5000, 4),
    (33, 3000, 2900, 260), (700, 100, 300, 90), (512, 4000, 2048, 16), (257, 130, 127, 129)])
def test_window_and_sinks(kind, paged, tokens, past, window, sinks):
    """The rows of the past that are neither sinks nor in the first token's window are not-a-numbers, and pages without a
    visible row have no valid name."""
    p = Prompt(kind, past + tokens, window=window, sinks=sinks, paged=paged)
    p.fill(past)
    p.chunk(tokens)


@KINDS
@pytest.mark.parametrize("tokens,past,window,sinks", [(300, 0, 0, 0), (200, 1500, 0, 0), (400, 900, 200, 5)])
def test_fp32_activations(kind, tokens, past, window, sinks):
    for paged in (False, True):
        p = Prompt(kind, past + tokens, window=window, sinks=sinks, paged=paged, dtype=K.DTYPE_F32)
        p.fill(past)
        p.chunk(tokens)


@KINDS
@pytest.mark.parametrize("dtype", [K.DTYPE_BF16, K.DTYPE_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("tokens,past,window,sinks,kv_heads,group", [
    (129, 1152, 0, 0, 4, 4), (130, 1270, 0, 0, 4, 4), (256, 1281, 0, 0, 4, 4), (255, 4001, 0, 0, 4, 4), (200, 3000, 1280, 4, 4, 4),
    (131, 3000, 1290, 140, 4, 4), (100, 1500, 0, 0, 8, 4), (128, 2000, 1400, 33, 16, 2), (90, 1500, 0, 0, 4, 9), (201, 1500, 0, 0, 3, 5),
    (200, 1700, 1500, 7, 1, 16)])
def test_two_tiles_and_many_keys(kind, paged, dtype, tokens, past, window, sinks, kv_heads, group):
    """Chunks whose items are cut into two or four shares, or whose heads are too many for four."""
    p = Prompt(kind, past + tokens, kv_heads=kv_heads, group=group, window=window, sinks=sinks, paged=paged, dtype=dtype)
    p.fill(past)
    p.chunk(tokens)


@KINDS
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 3), (1, 8), (3, 2), (8, 2)])
def test_head_layouts(kind, kv_heads, group):
    for tokens, past, window, sinks in ((200, 0, 0, 0), (150, 900, 140, 6)):
        p = Prompt(kind, past + tokens, kv_heads=kv_heads, group=group, window=window, sinks=sinks)
        p.fill(past)
        p.chunk(tokens)


@KINDS
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
def test_a_prompt_in_chunks_and_then_tokens(kind, paged):
    """The operators together as a server runs them: a prompt in ragged chunks, then generated tokens by the single-token
    call, on one cache; every call's output and cache bytes are the model's."""
    from test_kv_decode_gpu import tolerance as token_tolerance

    p = Prompt(kind, 700, window=100, sinks=4, paged=paged)
    p.fill(0)
    for tokens in (5, 128, 300, 17, 1, 100):
        p.chunk(tokens)
    stream = torch.cuda.current_stream()
    workspace = torch.empty(K.kv_decode_workspace_bytes(), device="cuda", dtype=torch.uint8)
    for step in range(20):
        seed, position = 5000 + 10 * step, p.past
        (query, q), (gate, g) = (activation(normal(seed + i, 1, 16, D), K.DTYPE_BF16) for i in range(2))
        (key, k), (value, v) = (activation(normal(seed + 2 + i, 1, 4, D) * 2.0 ** (step % 4), K.DTYPE_BF16) for i in range(2))
        output = torch.empty(1, 16, D, device="cuda", dtype=torch.bfloat16)
        where = torch.tensor([position], device="cuda", dtype=torch.int32)
        rest = (where, 1, 16, 4, p.window, p.sinks, K.DTYPE_BF16, kind, workspace, workspace.numel(), stream)
        if paged:
            K.kv_paged_decode(query, key, value, gate, output, p.cache, p.pool_pages, p.table(1), p.capacity // PAGE, *rest)
        else:
            K.kv_batched_decode(query, key, value, gate, output,
                                torch.tensor([p.cache.data_ptr()], device="cuda"),
                                torch.tensor([p.capacity], device="cuda", dtype=torch.int32), *rest)
        p.model.store(position, np.stack([k[0].numpy(), v[0].numpy()])[:, :, None])
        p.past += 1
        torch.cuda.synchronize()
        out, size, spread, total = attention(p.model, q, g, position, p.window, p.sinks)
        assert ((output.double() - out).abs() <= token_tolerance(out, size, spread, total, torch.bfloat16)).all()
        p.check_cache()
    assert K.device_status(stream) == 0


@KINDS
@pytest.mark.parametrize("dtype", [K.DTYPE_BF16, K.DTYPE_F32], ids=["bf16", "f32"])
def test_calls_one_behind_the_other_without_waiting(kind, dtype):
    """Chunks and tokens enqueued on one stream with nothing between them, one workspace for all: outputs and the cache are
    those of the same calls made one at a time."""
    heads, window, sinks, capacity = 16, 150, 5, 600
    stream = torch.cuda.current_stream()
    chunks, total = [130, 17, 200, 1, 60], 408
    new = [normal(i, total + 20, h, D).cuda().to(torch.float32 if dtype == K.DTYPE_F32 else torch.bfloat16)
           for i, h in ((1, heads), (2, 4), (3, 4), (4, heads))]
    scratch = torch.empty(1 << 22, device="cuda", dtype=torch.uint8)
    capacities = torch.tensor([capacity], device="cuda", dtype=torch.int32)
    positions = [torch.tensor([total + i], device="cuda", dtype=torch.int32) for i in range(20)]

    def calls(wait):
        cache = to_device(Cache(kind, 4, capacity).bytes)
        pointer = torch.tensor([cache.data_ptr()], device="cuda")
        output = torch.zeros_like(new[0])
        torch.cuda.synchronize()
        past = 0
        for tokens in chunks:
            rows = slice(past, past + tokens)
            shape = K.Qwen35AttentionShape(tokens, heads, 4, D, capacity, past)
            K.kv_attention_prefill(*[t[rows] for t in new], output[rows], cache, cache.numel() * cache.element_size(), scratch,
                                   scratch.numel(), shape, window, sinks, dtype, kind, stream)
            past += tokens
            if wait:
                torch.cuda.synchronize()
        for i in range(20):
            rows = slice(past + i, past + i + 1)
            K.kv_batched_decode(*[t[rows] for t in new], output[rows], pointer, capacities, positions[i], 1, heads, 4, window,
                                sinks, dtype, kind, scratch, scratch.numel(), stream)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert K.device_status(stream) == 0
        return output, cache

    (one, cache_one), (other, cache_other) = calls(True), calls(False)
    assert torch.equal(cache_one, cache_other)
    # (a prompt's sums do not depend on timing, a token's neither)
    assert torch.equal(one, other) and torch.isfinite(one.float()).all()


@KINDS
def test_a_long_prompt_behind_a_window(kind):
    p = Prompt(kind, 6000, kv_heads=2, group=2, window=700, sinks=130)
    p.fill(0)
    p.chunk(4100)
    p.chunk(1900)


def test_a_page_outside_the_pool_is_flagged_and_not_touched():
    p = Prompt(K.KV_E4M3, 600, paged=True)
    p.fill(300)
    p.order[1] = p.pool_pages + 9
    before = p.cache.clone()
    p.chunk(100, check=False)
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == K.DEVICE_PAGE_OUT_OF_RANGE
    assert torch.equal(before, p.cache)  # rows 300 .. 399 belong to the page that is not there


@KINDS
def test_captured_and_replayed(kind):
    stream = torch.cuda.current_stream()
    p = Prompt(kind, 900, window=200, sinks=3)
    p.fill(500)
    graph = torch.cuda.CUDAGraph()
    heads, tokens = 16, 300
    query, key, value, gate = (normal(i, tokens, h, D).cuda().bfloat16() for i, h in ((1, 16), (2, 4), (3, 4), (4, 16)))
    output = torch.zeros(tokens, heads, D, device="cuda", dtype=torch.bfloat16)
    shape = K.Qwen35AttentionShape(tokens, heads, 4, D, p.capacity, p.past)
    need = K.kv_prefill_workspace_bytes(shape, p.window, p.sinks, kind)
    workspace = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)
    call = lambda: K.kv_attention_prefill(query, key, value, gate, output, p.cache,
                                          p.cache.numel() * p.cache.element_size(), workspace, need, shape, p.window,
                                          p.sinks, K.DTYPE_BF16, kind, stream)
    call()
    torch.cuda.synchronize()
    eager = output.clone()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for _ in range(2):
        output.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(output, eager)
