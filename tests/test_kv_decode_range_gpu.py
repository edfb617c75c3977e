"""Single-token attention over rows of very different magnitudes and over rows with infinities, against a plain 64-bit model."""
import math

import numpy as np
import pytest
import torch

from raftinfer_b200 import kernels as K
from kv_util import BLOCK, D, HALF_STEP, Cache, activation, from_device, normal, scale_for, visible
from test_kv_decode_gpu import PARTS, Batch

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [K.DTYPE_F32, K.DTYPE_BF16], ids=["f32", "bf16"])


def store_blocks(cache, rows):
    """Cache.store(0, rows) of finite rows, all blocks at once."""
    if not cache.eight_bit:
        cache.store(0, rows.numpy())
        return
    n = rows.shape[2]
    blocks = -(-n // BLOCK)
    x = torch.zeros(2, cache.kv_heads, blocks * BLOCK, D)
    x[:, :, :n] = rows
    x = x.view(2, cache.kv_heads, blocks, BLOCK * D)
    scale = torch.from_numpy(np.vectorize(scale_for, otypes=[np.float64])(x.abs().amax(-1).double().numpy()))
    codes = (x.double() / scale[..., None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8)
    record = cache.bytes[:, :, :blocks]
    record[..., :n * D if blocks == 1 else BLOCK * D] = codes[..., :n * D if blocks == 1 else BLOCK * D].numpy()
    record[..., BLOCK * D:BLOCK * D + 4] = scale.float().numpy()[..., None].view(np.uint8)


class Rows(Batch):
    """A batch whose queries have 8 in dim 0, so that a key's dim 0 sets its logit in every head, and whose rows are edited:
    edit(i, keys, values) changes rows [kv_heads, length, 256] of sequence i in place, the new token's (the last) among them."""

    def __init__(self, kind, lengths, dtype, seed, edit, **more):
        super().__init__(kind, lengths, dtype, seed, **more, poison=False)
        self.q[..., 0] = 8.0
        self.query, self.q = activation(self.q, dtype)
        for i, length in enumerate(lengths):
            rows = torch.cat([normal(seed + 10 + i, 2, self.kv_heads, length - 1, D),
                              torch.stack([self.k[i], self.v[i]])[:, :, None]], 2)
            rows[0, :, :, 0] = 0.0
            edit(i, rows[0], rows[1])
            self.k[i], self.v[i] = rows[0, :, -1], rows[1, :, -1]
            cache = Cache(kind, self.kv_heads, self.before[i].capacity)
            if length > 1:
                store_blocks(cache, rows[:, :, :-1])
            self.before[i], self.after[i] = cache, cache.copy()
        self.key, self.k = activation(self.k, dtype)
        self.value, self.v = activation(self.v, dtype)
        for i, length in enumerate(lengths):
            self.after[i].store(length - 1, np.stack([self.k[i].numpy(), self.v[i].numpy()])[:, :, None])
        if self.paged:
            self._place_pages(seed)
        else:
            for device, cache in zip(self.caches, self.before):
                bits = cache.bytes.view(np.int16) if cache.bytes.dtype == np.uint16 else cache.bytes
                device.copy_(torch.from_numpy(bits))

    def check_range(self):
        """Every sequence against the definition.  A logit is off by 2^-16 of sum |q k| / 16 and as much again for 32-bit sums, a
        weight by twice its logit's error (numerator and denominator) and 2^-16 a part, as in the tests of ordinary rows.  A
        weight over 8-bit rows is, times its block's scale, also off by 2^-40 of twice the largest such product of the head, and
        a code is at most 448.  Where the definition gives an infinity or a not-a-number, so does the call."""
        torch.cuda.synchronize()
        assert K.device_status(torch.cuda.current_stream()) == 0
        for i, length in enumerate(self.lengths):
            tokens = np.array(visible(length - 1, self.window, self.sinks))
            keys, values = self.after[i].values(tokens).repeat_interleave(self.group, 1).cuda()
            q = self.q[i].cuda().double()
            logits = (q[:, None] * keys).sum(-1) / 16.0
            weights = torch.softmax(logits, -1)
            gates = torch.sigmoid(self.g[i].cuda().double())
            out = (weights[..., None] * values).sum(1) * gates
            clean_k, clean_v = torch.nan_to_num(keys, 0, 0, 0), torch.nan_to_num(values, 0, 0, 0)
            spread = (q.abs()[:, None] * clean_k.abs()).sum(-1).amax(-1)[:, None] / 16.0
            size = (weights.nan_to_num(0)[..., None] * clean_v.abs()).sum(1) * gates
            limit = size * (4 * PARTS * spread + 4 * PARTS) + out.abs() * HALF_STEP[self.output.dtype] + 1e-37
            if self.kind == K.KV_E4M3:
                record = np.ascontiguousarray(self.after[i].bytes[1, :, tokens // BLOCK, BLOCK * D:BLOCK * D + 4])
                scale = torch.from_numpy(record.view(np.float32)[..., 0].T.copy()).cuda().double()
                product = (weights * scale.repeat_interleave(self.group, 0)).amax(-1)[:, None]
                limit = limit + len(tokens) * 2.0 ** -40 * 2.0 * 448.0 * product * gates
            got = self.output[i].double()
            assert torch.equal(torch.isnan(got), torch.isnan(out)), i
            infinite = torch.isinf(out)
            assert torch.equal(got[infinite], out[infinite]), i
            finite = torch.isfinite(out)
            off = ((got - out).abs() / limit)[finite]
            assert off.numel() == 0 or float(off.max()) <= 1.0, (i, length, float(off.max()))
        self.check_caches()

    def check_caches(self):
        """Byte for byte, but for the bits of a not-a-number."""
        def same(got, want):
            got = from_device(got, want)
            if got.dtype == np.uint16:
                got, want = [np.where(x & 0x7FFF > 0x7F80, np.uint16(0x7FC0), x) for x in (got, want)]
            return np.array_equal(got, want)

        if self.paged:
            assert same(self.pool, self.want_pool)
        else:
            assert all(same(cache, want.bytes) for cache, want in zip(self.caches, self.after))


# Rows long and many enough for a warp to have several blocks of one.
MANY = [33, 70] + [1000 + 23 * i for i in range(20)]


def test_the_blocks_are_the_models():
    rows = normal(1, 2, 2, 45, D) * torch.exp(normal(2, 2, 2, 45, 1) * 9.0)
    one, other = Cache(K.KV_E4M3, 2, 64), Cache(K.KV_E4M3, 2, 64)
    one.store(0, rows[:, :, :32].numpy())
    store_blocks(other, rows[:, :, :32])
    assert np.array_equal(one.bytes, other.bytes)
    store_blocks(other, rows)
    one.store(32, rows[:, :, 32:].numpy())
    assert torch.equal(one.values(range(45)), other.values(range(45)))


@DTYPES
@pytest.mark.parametrize("power,where", [(45, "first"), (110, "first"), (45, "middle"), (30, "newest")])
def test_values_of_another_magnitude_without_weight(dtype, power, where):
    """A block (of a warp's share the first, or one further on, or the new token) whose values are 2^power times the others' and
    whose weight is e^-100 or e^-120: what the others hold counts."""
    def edit(i, keys, values):
        n = keys.shape[1]
        at = {"first": slice(0, 64), "middle": slice(n // 32 * 16, n // 32 * 16 + 16), "newest": slice(n - 1, n)}[where]
        keys[:, at, 0] = -200.0 if power < 100 else -240.0
        values[:, at] *= 2.0 ** power

    b = Rows(K.KV_E4M3, MANY, dtype, 200 + power, edit, paged=where == "middle")
    b.run()
    b.check_range()


@DTYPES
@pytest.mark.parametrize("group", [1, 4])
def test_products_of_weights_and_values_that_balance(dtype, group):
    """Blocks whose weights fall by e^-7 (2^-10) as their values grow by 2^10, and the reverse: all of them count."""
    def falling(i, keys, values):
        for b in range(keys.shape[1] // 16):
            step = min(b // 4, 8)
            keys[:, 16 * b:16 * b + 16, 0] = -14.0 * step
            values[:, 16 * b:16 * b + 16] *= 2.0 ** (10 * step)

    def rising(i, keys, values):
        for b in range(keys.shape[1] // 16):
            step = min(b // 4, 8)
            keys[:, 16 * b:16 * b + 16, 0] = 14.0 * step
            values[:, 16 * b:16 * b + 16] *= 2.0 ** (-10 * step)

    for edit in (falling, rising):
        b = Rows(K.KV_E4M3, MANY, dtype, 230, edit, group=group)
        b.run()
        b.check_range()


@DTYPES
def test_a_block_whose_large_rows_are_outside_the_window(dtype):
    def edit(i, keys, values):
        low = max(0, keys.shape[1] - 600)
        values[:, low // 16 * 16:low] *= 2.0 ** 40

    b = Rows(K.KV_E4M3, MANY, dtype, 240, edit, window=600, sinks=0)
    b.run()
    b.check_range()


def test_magnitudes_at_the_ends_of_the_scales():
    """Values around 2^119 without weight beside values around 2^-90, logits in the hundreds."""
    def edit(i, keys, values):
        keys[:, :64, 0] = -440.0
        values[:, :64] = values[:, :64].clamp(-1, 1) * 2.0 ** 119
        keys[:, 64:, 0] = 400.0
        values[:, 64:] *= 2.0 ** -90

    b = Rows(K.KV_E4M3, [100, 800] + MANY, K.DTYPE_F32, 250, edit)
    b.run()
    b.check_range()


LENGTHS = [33, 700, 1, 3001, 18]


@DTYPES
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("kv_heads,group", [(2, 4), (2, 3), (1, 1)])
def test_keys_that_are_infinite(dtype, paged, kv_heads, group):
    """A logit of minus infinity is a weight of zero; one of plus infinity makes its heads not-a-numbers."""
    def edit(i, keys, values):
        n = keys.shape[1]
        if n > 1:
            keys[:, n // 2, 0] = -math.inf
            keys[:, 0, 0] = -math.inf
        if n == 700:
            keys[:, n - 1, 0] = -math.inf
        if n == 18:
            keys[0, 3, 0] = math.inf

    b = Rows(K.KV_BF16, LENGTHS, dtype, 260, edit, kv_heads=kv_heads, group=group, paged=paged)
    b.run()
    b.check_range()
    assert torch.isfinite(b.output[:4].float()).all() and torch.isnan(b.output[4, 0].float()).all()


@DTYPES
@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("lengths", [LENGTHS, [40 + 13 * i for i in range(30)]], ids=["few", "many"])
def test_values_that_are_infinite(dtype, paged, lengths):
    """An infinity in a dim makes that dim's output infinite, two of unlike sign or a not-a-number a not-a-number, no other."""
    def edit(i, keys, values):
        n = keys.shape[1]
        values[:, n // 2, 5] = math.inf
        values[:, n - 1, 9] = -math.inf
        values[:, 0, 200], values[:, n // 3, 200] = math.inf, -math.inf
        values[0, n // 4, 255] = math.nan
        if n > 1:
            keys[:, n // 4, 0] = -math.inf

    b = Rows(K.KV_BF16, lengths, dtype, 270, edit, kv_heads=2, paged=paged)
    b.run()
    b.check_range()


@DTYPES
@pytest.mark.parametrize("lengths", [LENGTHS, [40 + 53 * i for i in range(30)]], ids=["few", "many"])
def test_an_infinite_value_under_a_weight_that_32_bits_do_not_hold(dtype, lengths):
    """A weight of e^-150 is not zero: in front of the tokens that have all of the weight, behind them, and in the new token."""
    def edit(i, keys, values):
        n = keys.shape[1]
        for at, dim in ((0, 3), (n // 2, 4), (n - 1, 5)):
            keys[:, at, 0], values[:, at, dim] = -300.0, math.inf
        values[:, n // 3, 5] = -math.inf

    b = Rows(K.KV_BF16, lengths, dtype, 290, edit, kv_heads=2)
    b.run()
    b.check_range()


@DTYPES
def test_infinities_that_the_window_hides(dtype):
    def edit(i, keys, values):
        n = keys.shape[1]
        for hidden in range(5, n - 50):
            keys[:, hidden, 0], values[:, hidden, 3] = math.inf, -math.inf
        values[:, n - 10, 4] = math.inf

    b = Rows(K.KV_BF16, [700, 77, 300], dtype, 280, edit, kv_heads=1, window=50, sinks=5)
    b.run()
    b.check_range()


@pytest.mark.parametrize("kind", [K.KV_BF16, K.KV_E4M3], ids=["bf16", "e4m3"])
def test_one_long_context_among_short_ones(kind):
    """Too many rows to cut each by itself: the long one's rows are put together from dozens of parts."""
    b = Rows(kind, [500] * 6 + [30001] + [500 + 7 * i for i in range(13)], K.DTYPE_F32, 300, lambda i, keys, values: None, kv_heads=2)
    b.run()
    b.check_range()
