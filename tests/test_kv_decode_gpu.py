"""Single-token attention over BF16 and 8-bit caches, whole and windowed, against a plain 64-bit model."""
import numpy as np
import pytest
import torch

from raftinfer_b200 import kernels as K
from kv_util import (D, HALF_STEP, PAGE, Cache, activation, attention, from_device, normal, to_device, visible)

pytestmark = pytest.mark.gpu

# Queries and weights are held as two parts of a 16-bit type, together 2^-16 of the value or less; a logit is then off by at
# most 2^-16 of sum |q k| / 16 (and 2^-16 of that for FP32 sums of 256 products), a weight by 2^-16 and twice its logit's
# error (numerator and denominator).
PARTS = 2.0 ** -16


# Weights over 8-bit rows are FP16 parts of weight / largest weight * scale / largest scale * 2^15, off by half of FP16's smallest
# step, 2^-25, as well: 2^-40 code * largest scale for each token of the sum.  The block with the largest scale has a value
# of 224 scales or more and a code is at most 448, so that is 2^-40 * 2 * max |v| for each token.
SMALLEST = 2.0 ** -40


def tolerance(out, size, spread, total, dtype):
    return size * (2 * 2 * PARTS * spread + 4 * PARTS) + SMALLEST * total + out.abs() * HALF_STEP[dtype] + 1e-30


class Batch:
    """Sequences with `lengths` tokens, the last of which the call under test brings; entries of length 0 are padding."""

    def __init__(self, kind, lengths, dtype, seed, kv_heads=4, group=4, window=0, sinks=0, paged=False, magnitude=None,
                 poison=True):
        self.kind, self.lengths, self.dtype, self.paged = kind, lengths, dtype, paged
        self.kv_heads, self.group, self.window, self.sinks = kv_heads, group, window, sinks
        heads, n = kv_heads * group, len(lengths)
        self.query, self.q = activation(normal(seed, n, heads, D), dtype)
        self.gate, self.g = activation(normal(seed + 1, n, heads, D), dtype)
        self.key, self.k = activation(normal(seed + 2, n, kv_heads, D), dtype)
        self.value, self.v = activation(normal(seed + 3, n, kv_heads, D), dtype)
        if magnitude is not None:
            self.value, self.v = activation(self.v * magnitude, dtype)
        self.before = []
        for i, length in enumerate(lengths):
            capacity = max(PAGE, -(-length // PAGE) * PAGE) if paged else max(1, length + (i % 3) * 7)
            cache = Cache(kind, kv_heads, capacity)
            if length > 1:
                cache.store(0, normal(seed + 10 + i, 2, kv_heads, length - 1, D).numpy())
                if poison and window:
                    seen = set(visible(length - 1, window, sinks))
                    cache.poison([t for t in range(length - 1) if t not in seen])
            self.before.append(cache)
        self.after = [c.copy() for c in self.before]
        for i, length in enumerate(lengths):
            if length:
                self.after[i].store(length - 1, np.stack([self.k[i].numpy(), self.v[i].numpy()])[:, :, None])
        self.positions = [length - 1 if length else K.NO_POSITION for length in lengths]
        self.output = torch.full((n, heads, D), 7.0, device="cuda", dtype=self.query.dtype)
        self.workspace = torch.full((K.kv_decode_workspace_bytes(),), 0xFF, device="cuda", dtype=torch.uint8)  # not-a-numbers
        self.device_positions = torch.from_numpy(np.array(self.positions, dtype=np.uint32).view(np.int32)).cuda()
        if paged:
            self._place_pages(seed)
        else:
            self.caches = [to_device(c.bytes) for c in self.before]
            self.pointers = torch.tensor([c.data_ptr() for c in self.caches], device="cuda", dtype=torch.int64)
            self.capacities = torch.tensor([c.capacity for c in self.before], device="cuda", dtype=torch.int32)

    def _place_pages(self, seed):
        used = [c.capacity // PAGE for c in self.before]
        self.pool_pages = sum(used) + 2
        order = np.random.default_rng(seed).permutation(self.pool_pages)
        shape = (self.pool_pages, *self.before[0].pages().shape[1:])
        pool = np.full(shape, 0x7F if self.kind == K.KV_E4M3 else 0x7FC1, dtype=self.before[0].bytes.dtype)
        self.want_pool = pool.copy()
        tables = np.full((len(used), max(used)), 0xFFFFFFFF, dtype=np.uint32)
        at = 0
        for i, n in enumerate(used):
            mine = order[at:at + n]
            at += n
            pool[mine], self.want_pool[mine] = self.before[i].pages(), self.after[i].pages()
            seen = {t // PAGE for t in visible(self.lengths[i] - 1, self.window, self.sinks)} if self.lengths[i] else set()
            for b in seen:  # pages that are not visible have no valid name
                tables[i, b] = mine[b]
        self.tables, self.pool = torch.from_numpy(tables.view(np.int32)).cuda(), to_device(pool)
        self.max_blocks = max(used)

    def run(self, stream=None, workspace=None, window=None):
        stream = stream or torch.cuda.current_stream()
        workspace = self.workspace if workspace is None else workspace
        common = (len(self.lengths), self.kv_heads * self.group, self.kv_heads, self.window if window is None else window,
                  self.sinks, self.dtype, self.kind, workspace, workspace.numel(), stream)
        if self.paged:
            K.kv_paged_decode(self.query, self.key, self.value, self.gate, self.output, self.pool, self.pool_pages,
                              self.tables, self.max_blocks, self.device_positions, *common)
        else:
            K.kv_batched_decode(self.query, self.key, self.value, self.gate, self.output, self.pointers, self.capacities,
                                self.device_positions, *common)

    def check(self, outputs=None):
        got = (self.output if outputs is None else outputs).double()
        for i, length in enumerate(self.lengths):
            if not length:
                assert (got[i] == 7.0).all(), "padding was written"
                continue
            out, size, spread, total = attention(self.after[i], self.q[i:i + 1], self.g[i:i + 1], length - 1, self.window, self.sinks)
            off = (got[i:i + 1] - out).abs()
            limit = tolerance(out, size, spread, total, self.output.dtype)
            assert (off <= limit).all(), (i, length, float((off / limit).max()))
        self.check_caches()

    def check_caches(self):
        if self.paged:
            assert np.array_equal(from_device(self.pool, self.want_pool), self.want_pool)
        else:
            for cache, want in zip(self.caches, self.after):
                assert np.array_equal(from_device(cache, want.bytes), want.bytes)


KINDS = pytest.mark.parametrize("kind", [K.KV_BF16, K.KV_E4M3], ids=["bf16", "e4m3"])
LENGTHS = [1, 2, 15, 16, 17, 33, 128, 129, 255, 256, 257, 1000, 1025, 3001]


@KINDS
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("dtype", [K.DTYPE_F32, K.DTYPE_BF16], ids=["f32", "bf16"])
def test_whole_context_at_every_length(kind, paged, dtype):
    b = Batch(kind, LENGTHS, dtype, 11, paged=paged)
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    b.check()


@KINDS
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 16), (17, 0), (100, 20), (256, 4), (256, 300),
                                          (1000, 257), (4096, 8)])
def test_window_and_sinks(kind, paged, window, sinks):
    """Rows outside the window hold not-a-numbers, and pages without a visible row have no valid name."""
    b = Batch(kind, LENGTHS, K.DTYPE_F32, 29, window=window, sinks=sinks, paged=paged)
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    b.check()


@KINDS
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (3, 2), (2, 3), (8, 4), (5, 1)])
def test_head_layouts(kind, kv_heads, group):
    for paged in (False, True):
        b = Batch(kind, [700, 1, 33], K.DTYPE_F32, 5, kv_heads=kv_heads, group=group, paged=paged)
        b.run()
        torch.cuda.synchronize()
        b.check()


@KINDS
def test_one_long_context(kind):
    for length, window in ((40001, 0), (40001, 20000)):
        b = Batch(kind, [length], K.DTYPE_F32, 3, kv_heads=2, window=window, sinks=5 if window else 0)
        b.run()
        torch.cuda.synchronize()
        b.check()


@KINDS
def test_a_batch_with_padding_and_a_ragged_many(kind):
    lengths = [0, 5, 0, 900, 16, 0] + [1 + (37 * i) % 300 for i in range(150)] + [0]
    b = Batch(kind, lengths, K.DTYPE_BF16, 7, kv_heads=1, group=2, paged=True)
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    b.check()


def test_nothing_but_padding_leaves_everything():
    b = Batch(K.KV_E4M3, [0, 0], K.DTYPE_BF16, 7)
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    b.check()


def test_scales_follow_magnitudes_token_by_token():
    """Forty tokens one by one, of magnitudes from 2^-40 to 2^40 and zeros: every step's cache bytes are the model's, and
    rows in front are rounded again only when a scale grows."""
    magnitudes = [1.0, 2.0 ** -40, 0.0, 3.0, 2.0 ** 10, 1e-3, 5.0, 2.0 ** 20] * 5
    caches, stream = None, torch.cuda.current_stream()
    for step, magnitude in enumerate(magnitudes):
        b = Batch(K.KV_E4M3, [step + 1], K.DTYPE_F32, 100 + step, kv_heads=2, group=1, magnitude=magnitude)
        if caches is None:
            cache = Cache(K.KV_E4M3, 2, 64)
            caches, capacity = to_device(cache.bytes), torch.tensor([64], device="cuda", dtype=torch.int32)
            pointer = torch.tensor([caches.data_ptr()], device="cuda")
        cache.store(step, np.stack([b.k[0].numpy(), b.v[0].numpy()])[:, :, None])
        b.pointers, b.capacities, b.caches, b.after = pointer, capacity, [caches], [cache]
        b.run()
        torch.cuda.synchronize()
        b.check()
    assert K.device_status(stream) == 0


def test_values_at_the_ends_of_the_range():
    """The largest and smallest FP32 numbers: the scale is held between 2^-100 and 2^119."""
    for magnitude in (2.0 ** 125, 2.0 ** -130, 2.0 ** -99):
        b = Batch(K.KV_E4M3, [16, 17], K.DTYPE_F32, 41, kv_heads=1, group=2, magnitude=magnitude)
        b.run()
        torch.cuda.synchronize()
        b.check_caches()
        assert torch.isfinite(b.output).all()


def test_infinities_saturate_and_not_a_number_stays():
    b = Batch(K.KV_E4M3, [20], K.DTYPE_F32, 43, kv_heads=1, group=1)
    b.value[0, 0, 3], b.value[0, 0, 4], b.value[0, 0, 5] = float("inf"), -float("inf"), float("nan")
    b.after[0] = b.before[0].copy()
    b.after[0].store(19, np.stack([b.k[0].numpy(), b.value[0].cpu().numpy()])[:, :, None])
    b.run()
    torch.cuda.synchronize()
    b.check_caches()
    assert torch.isnan(b.output[0, 0]).nonzero().flatten().tolist() == [5]


@KINDS
def test_logits_that_are_far_apart(kind):
    """Queries thirty times larger: a few keys take all of the weight, and running maxima move by hundreds."""
    b = Batch(kind, [1500, 40], K.DTYPE_F32, 47)
    b.query, b.q = activation(b.q * 30.0, K.DTYPE_F32)
    b.run()
    torch.cuda.synchronize()
    b.check()


@KINDS
def test_positions_outside_a_cache_are_flagged_and_skipped(kind):
    b = Batch(kind, [40, 300, 17], K.DTYPE_BF16, 51)
    b.device_positions[0] = b.before[0].capacity
    b.after[0] = b.before[0]
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == K.DEVICE_POSITION_OUT_OF_RANGE
    assert (b.output[0] == 7.0).all()
    b.lengths[0] = 0
    b.check()


@KINDS
def test_a_page_outside_the_pool_is_flagged_and_not_touched(kind):
    for bad_block, lengths in ((0, [300, 700]), (1, [300, 700])):  # a page that is read, and the one that is written
        b = Batch(kind, lengths, K.DTYPE_BF16, 53, paged=True)
        b.tables[0, bad_block] = b.pool_pages + 5
        b.run()
        torch.cuda.synchronize()
        assert K.device_status(torch.cuda.current_stream()) == K.DEVICE_PAGE_OUT_OF_RANGE
        out, size, spread, total = attention(b.after[1], b.q[1:2], b.g[1:2], lengths[1] - 1, 0, 0)
        assert ((b.output[1:2].double() - out).abs() <= tolerance(out, size, spread, total, torch.bfloat16)).all()


def test_a_cache_pointer_off_its_boundary_is_flagged_and_not_read():
    b = Batch(K.KV_E4M3, [40, 300], K.DTYPE_BF16, 57)
    b.pointers[0] += 4
    b.after[0] = b.before[0]
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == K.DEVICE_POINTER_MISALIGNED
    assert (b.output[0] == 7.0).all()
    b.lengths[0] = 0
    b.check()


@KINDS
def test_a_null_cache_pointer_is_flagged_and_not_read(kind):
    b = Batch(kind, [40, 300, 0], K.DTYPE_BF16, 59)
    b.pointers[0] = 0
    b.pointers[2] = 0  # beside padding a pointer may be anything
    b.after[0] = b.before[0]
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == K.DEVICE_POINTER_MISALIGNED
    assert (b.output[0] == 7.0).all()
    b.lengths[0] = 0
    b.check()
    b.pointers[0] = b.caches[0].data_ptr()
    b.device_positions[0] = -1  # padding
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0


@KINDS
def test_captured_steps_that_share_a_workspace(kind):
    """Two steps of different batches in one graph each, one workspace, replayed in turn."""
    stream = torch.cuda.current_stream()
    batches = [Batch(kind, [700, 33], K.DTYPE_BF16, 61, paged=True), Batch(kind, [2000], K.DTYPE_BF16, 67)]
    shared = batches[0].workspace
    graphs = []
    for b in batches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            b.run(stream, shared)
        graphs.append(graph)
    for _ in range(3):
        for b, graph in zip(batches, graphs):
            b.output.fill_(7.0)
            graph.replay()
    torch.cuda.synchronize()
    assert K.device_status(stream) == 0
    for b in batches:
        b.check()


@KINDS
def test_a_captured_step_with_positions_that_move(kind):
    """One graph, replayed with the token and its position rewritten in place: a context that grows from 250 to 262 tokens
    (over a block and over a page) behind a window, beside an entry that turns into padding."""
    stream, window, sinks = torch.cuda.current_stream(), 40, 3
    b = Batch(kind, [250, 20], K.DTYPE_F32, 97, window=window, sinks=sinks, paged=True, poison=False)
    pages = torch.arange(4, dtype=torch.int32)  # two pages a sequence
    before = [Cache(kind, 4, 512), Cache(kind, 4, 512)]
    for i, n in ((0, 249), (1, 19)):
        before[i].store(0, normal(500 + i, 2, 4, n, D).numpy())
    b.pool = to_device(np.concatenate([c.pages() for c in before]))
    b.tables, b.pool_pages, b.max_blocks = pages.view(2, 2).cuda(), 4, 2
    graph, first = torch.cuda.CUDAGraph(), True
    for step in range(12):
        for t, x in ((b.query, b.q), (b.key, b.k), (b.value, b.v), (b.gate, b.g)):
            x.copy_(normal(1000 + 10 * step + x.shape[1], *x.shape))
            t.copy_(x)
        position = [249 + step, 19 + step if step < 5 else K.NO_POSITION]
        b.device_positions.copy_(torch.from_numpy(np.array(position, dtype=np.uint32).view(np.int32)))
        b.output.fill_(7.0)
        if first:
            b.run()  # what is captured has run once
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                b.run()
            first = False
        graph.replay()
        torch.cuda.synchronize()
        assert K.device_status(stream) == 0
        for i in range(2):
            if position[i] == K.NO_POSITION:
                assert (b.output[i] == 7.0).all()
                continue
            before[i].store(position[i], np.stack([b.k[i].numpy(), b.v[i].numpy()])[:, :, None])
            out, size, spread, total = attention(before[i], b.q[i:i + 1], b.g[i:i + 1], position[i], window, sinks)
            assert ((b.output[i:i + 1].double() - out).abs() <= tolerance(out, size, spread, total, torch.float32)).all()
        want = np.concatenate([c.pages() for c in before])
        assert np.array_equal(from_device(b.pool, want), want)


@KINDS
def test_pages_behind_four_gigabytes(kind):
    """A pool of more than 2^32 bytes, the sequence's pages at its end and its beginning."""
    page_bytes = K.kv_cache_bytes(4, PAGE, kind)
    pool_pages = (1 << 32) // page_bytes + 9
    b = Batch(kind, [600], K.DTYPE_F32, 103, paged=True)
    pool = torch.zeros(pool_pages, *b.pool.shape[1:], device="cuda", dtype=b.pool.dtype)
    where = torch.tensor([pool_pages - 1, 0, pool_pages - 3], device="cuda")
    pool[where] = b.pool[b.tables[0].long()]
    want = b.want_pool[b.tables[0].cpu().numpy()]
    b.pool, b.pool_pages, b.tables = pool, pool_pages, where.int()[None]
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    out, size, spread, total = attention(b.after[0], b.q, b.g, 599, 0, 0)
    assert ((b.output.double() - out).abs() <= tolerance(out, size, spread, total, torch.float32)).all()
    assert np.array_equal(from_device(pool[where], want), want)


@KINDS
def test_more_sequences_than_a_warp_has_lanes_for(kind):
    lengths = [1 + (7 * i) % 40 for i in range(1500)]
    lengths[3] = lengths[1111] = 0
    b = Batch(kind, lengths, K.DTYPE_BF16, 101, kv_heads=1, group=1)
    b.run()
    torch.cuda.synchronize()
    assert K.device_status(torch.cuda.current_stream()) == 0
    b.check()


@KINDS
def test_calls_on_two_streams_at_once(kind):
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    batches = [Batch(kind, [3000 + 100 * i, 5], K.DTYPE_BF16, 71 + i) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, stream in zip(batches, streams):
            b.run(stream)
    torch.cuda.synchronize()
    for b in batches:
        b.check()


@KINDS
def test_the_same_call_twice_gives_the_same_bits(kind):
    b = Batch(kind, LENGTHS, K.DTYPE_F32, 83)
    b.run()
    first = b.output.clone()
    b.run()
    torch.cuda.synchronize()
    assert torch.equal(first, b.output)
    b.check()
