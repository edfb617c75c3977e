"""A plain model of the BF16 and 8-bit KV caches and of attention over them, in 64 bits, for the tests of the kv_* calls."""
import math

import numpy as np
import torch

from raftinfer_b200 import kernels as K

D, PAGE, BLOCK, RECORD = 256, 256, 16, 4112
E4M3_VALUES = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
NAN_CODE = 0x7F


def scale_for(amax):
    """Least power of two s with amax <= 448 s, between 2^-100 and 2^119."""
    if amax == 0:
        return 2.0 ** -100
    e = math.frexp(amax)[1] - 12
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** min(119, max(-100, e))


_POSITIVE = E4M3_VALUES[:127]  # 0 .. 448, ascending


def codes_for(x):
    """Nearest e4m3 code of each value, ties to the even code; beyond 448 the largest, a not-a-number the code of one."""
    x = np.asarray(x, dtype=np.float64)
    magnitude = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    upper = np.searchsorted(_POSITIVE, magnitude).clip(0, 126)
    lower = np.maximum(upper - 1, 0)
    to_upper, to_lower = _POSITIVE[upper] - magnitude, magnitude - _POSITIVE[lower]
    pick = np.where(to_upper < to_lower, upper, np.where(to_lower < to_upper, lower, np.where(upper % 2 == 0, upper, lower)))
    code = (pick | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)
    return np.where(np.isnan(x), np.uint8(NAN_CODE), code)


class Cache:
    """One sequence's rows: [K, V][kv head][token].  What was never written is a not-a-number."""

    def __init__(self, kind, kv_heads, capacity):
        self.kind, self.kv_heads, self.capacity = kind, kv_heads, capacity
        self.eight_bit = kind == K.KV_E4M3
        if self.eight_bit:
            blocks = -(-capacity // BLOCK)
            self.bytes = np.full((2, kv_heads, blocks, RECORD), NAN_CODE, dtype=np.uint8)
        else:
            self.bytes = np.full((2, kv_heads, capacity, D), 0x7FC1, dtype=np.uint16)

    def store(self, past, rows):
        """rows [2, kv_heads, n, 256] (FP32 values) at tokens past .. past + n - 1."""
        n = rows.shape[2]
        if not self.eight_bit:
            bits = torch.from_numpy(np.ascontiguousarray(rows, dtype=np.float32)).to(torch.bfloat16).view(torch.int16)
            self.bytes[:, :, past:past + n] = bits.numpy().view(np.uint16)
            return
        for plane in range(2):
            for head in range(self.kv_heads):
                for block in range(past // BLOCK, (past + n - 1) // BLOCK + 1):
                    record = self.bytes[plane, head, block]
                    codes = record[:BLOCK * D].reshape(BLOCK, D)
                    first, last = max(past, block * BLOCK), min(past + n, (block + 1) * BLOCK)
                    new = rows[plane, head, first - past:last - past].astype(np.float64)
                    finite = np.abs(new[np.isfinite(new)])
                    scale, kept = scale_for(finite.max() if finite.size else 0.0), first - block * BLOCK
                    if kept:
                        before = float(record[BLOCK * D:BLOCK * D + 4].view(np.float32)[0])
                        if before > scale:
                            scale = before
                        elif scale > before:
                            codes[:kept] = codes_for(E4M3_VALUES[codes[:kept]] * (before / scale))
                    codes[kept:last - block * BLOCK] = codes_for(new / scale)
                    record[BLOCK * D:BLOCK * D + 4].view(np.float32)[0] = scale

    def values(self, tokens):
        """K and V of the tokens in 64 bits: [2, kv_heads, n, 256]."""
        tokens = np.asarray(tokens)
        if not self.eight_bit:
            bits = self.bytes[:, :, tokens].astype(np.uint32) << 16
            return torch.from_numpy(bits.view(np.float32).astype(np.float64))
        record = self.bytes[:, :, tokens // BLOCK]
        codes = record[..., :BLOCK * D].reshape(*record.shape[:3], BLOCK, D)
        picked = codes[:, :, np.arange(len(tokens)), tokens % BLOCK]
        scale = np.ascontiguousarray(record[..., BLOCK * D:BLOCK * D + 4]).view(np.float32).astype(np.float64)
        return torch.from_numpy(E4M3_VALUES[picked] * scale)

    def poison(self, tokens):
        """Rows that nothing may read."""
        for t in tokens:
            if self.eight_bit:
                self.bytes[:, :, t // BLOCK, (t % BLOCK) * D:(t % BLOCK + 1) * D] = NAN_CODE
            else:
                self.bytes[:, :, t] = 0x7FC1

    def pages(self):
        """The rows as pages [n][2][kv_heads][...]; the capacity is a multiple of 256."""
        n = self.capacity // PAGE
        per_page = self.bytes.shape[2] // n
        return self.bytes.reshape(2, self.kv_heads, n, per_page, -1).transpose(2, 0, 1, 3, 4)

    def copy(self):
        other = Cache(self.kind, self.kv_heads, self.capacity)
        other.bytes = self.bytes.copy()
        return other


def to_device(array):
    signed = array.view(np.int16) if array.dtype == np.uint16 else array
    return torch.from_numpy(np.ascontiguousarray(signed)).cuda()


def from_device(tensor, like):
    return tensor.cpu().numpy().view(like.dtype).reshape(like.shape)


def visible(position, window, sinks):
    low = max(0, position + 1 - window) if window else 0
    return list(range(min(sinks, low))) + list(range(low, position + 1))


def attention(cache, query, gate, past, window, sinks):
    """Rows query, gate [n, heads, 256] (FP32) at positions past .. in 64 bits: the output; attention of |v| times the gate,
    which bounds what relative errors of weights do; the largest sum |q_d k_d| / 16 of a visible key, which bounds what
    relative errors of products do to a logit; and the number of visible tokens times the head's largest |v| times two times the
    gate, which bounds what errors of weights relative to the largest one do."""
    n, heads, _ = query.shape
    group = heads // cache.kv_heads
    tokens = sorted(set().union(*[visible(past + i, window, sinks) for i in (0, n - 1)], range(past, past + n)))
    keys, values = cache.values(tokens).cuda()
    token, position = torch.tensor(tokens, device="cuda"), torch.arange(past, past + n, device="cuda")[:, None]
    seen = token <= position
    if window:
        seen &= (token > position - window) | (token < sinks)
    keys, values = keys.repeat_interleave(group, 0), values.repeat_interleave(group, 0)  # [heads, tokens, 256]
    q = query.cuda().double().permute(1, 0, 2)
    logits = (q @ keys.transpose(1, 2) / 16.0).masked_fill(~seen, -math.inf)
    weights = torch.softmax(logits, -1)
    held = seen.any(0)[:, None]
    clean = torch.where(held, values, torch.zeros_like(values))
    gates = torch.sigmoid(gate.cuda().double())
    out = (weights @ clean).permute(1, 0, 2) * gates
    size = (weights @ clean.abs()).permute(1, 0, 2) * gates
    spread = (q.abs() @ torch.where(held, keys, torch.zeros_like(keys)).abs().transpose(1, 2) / 16.0).masked_fill(~seen, 0.0)
    total = 2.0 * seen.sum(-1)[:, None, None] * clean.abs().amax((1, 2))[None, :, None] * gates
    return out, size, spread.amax(-1).permute(1, 0)[..., None], total


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def activation(x, dtype):
    """Device tensor of the activation type and the FP32 values it holds."""
    t = x.to(torch.float32 if dtype == K.DTYPE_F32 else torch.bfloat16)
    return t.cuda(), t.float()


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
