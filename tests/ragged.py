"""Plain 64-bit statements of the ragged-batch operators, and batches to try them on."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # a rounding is off by at most this, relative to the value


def rope_reference(x, w, eps, positions, inv_freq, rotary, factor=1.0):
    """x [T, H, 128] in 64 bits -> normed (w given) and turned rows."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    half = rotary // 2
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = (angle.cos() * factor)[:, None], (angle.sin() * factor)[:, None]
    a, b = x[..., :half], x[..., half:rotary]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rotary:]], -1)


def assert_rows_close(got, want, what=""):
    """fp16 rows of a norm and a rotation in 32 bits: half a step of fp16 (2^-25 below its normal range), and the 32-bit
    arithmetic: a sum of 128 squares in 8 + 4 roundings, a reciprocal root, two weights, cos / sin and two products, in all
    at most 32 roundings of 2^-24 of the two terms of a rotation, each at most the row's largest value."""
    want = want.double()
    tol = HALF_STEP[torch.float16] * want.abs() + 2.0 ** -25 + 2 * 32 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (err <= tol).all(), f"{what}: {int((err > tol).sum())} values off, worst {float((err / tol).max()):.2f} of the tolerance"


def attention_reference(q, k_pool, v_pool, pages, past, new, window=0, gate=None, scale=None):
    """(out, mean |v| under the same weights) in 64 bits for the rows of every sequence in order."""
    T, Hq, D = q.shape
    Hkv, P = k_pool.shape[1], k_pool.shape[2]
    G = Hq // Hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    t0 = 0
    for b, (a, n) in enumerate(zip(past, new)):
        if n == 0:
            continue
        pos = torch.arange(a + n, device=q.device)
        rows = a + torch.arange(n, device=q.device)
        seen = pos[None, :] <= rows[:, None]
        if window:
            seen &= pos[None, :] > rows[:, None] - window
        used = seen.any(0)  # pages below the window may have been given back
        ids = torch.where(used, pages[b, pos // P].long(), 0)
        for h in range(Hkv):
            k, v = (torch.where(used[:, None], x[ids, h, pos % P].double(), 0.0) for x in (k_pool, v_pool))
            s = torch.einsum("tgd,kd->tgk", q[t0:t0 + n, h * G:(h + 1) * G].double(), k) * (scale or 1 / math.sqrt(D))
            w = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            out[t0:t0 + n, h * G:(h + 1) * G] = w @ v
            size[t0:t0 + n, h * G:(h + 1) * G] = w @ v.abs()
        t0 += n
    if gate is not None:
        g = torch.nn.functional.softplus(gate[:t0].double())[..., None]
        out[:t0] *= g
        size[:t0] *= g
    return out, size


def assert_attention_close(got, want, size, keys, what=""):
    """Half a step of the output's type; half a step of fp16 for each weight (the probabilities enter the second product as
    fp16), which moves a row by at most 2^-11 of its mean |v|; for weights in fp16's subnormal range 2^-25 of the largest
    weight each, `keys` times at most; and 2^-14 of the mean |v| for the 32-bit scores (128 products of values of about 1,
    scaled, in the exponent), the exponential's 2^-22 and the sums.  A value below 2^-14 (a gate of e^-8, say) is a subnormal
    fp16: its steps are 2^-24, so the rounding is off by 2^-25 however small the value."""
    tol = HALF_STEP[got.dtype] * want.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0.0) + (2.0 ** -11 + 2.0 ** -14) * size + (keys * 2.0 ** -25 + 1e-7) * size.amax(-1, keepdim=True)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.numel()} values off, worst {float((err / tol).max()):.2f} of the tolerance"


class Batch:
    """Pools with cached and new tokens of several sequences in scattered pages; slots that no new token sees hold `filler`."""

    def __init__(self, device, past, new, Hq, Hkv, P=16, seed=0, filler=float("nan"), window=0, spare_rows=0, tight=True):
        g = torch.Generator(device=device).manual_seed(seed)
        self.past, self.new = list(past), list(new)
        need = [-(-(a + n) // P) for a, n in zip(past, new)]
        num_pages = sum(need) + 3
        ids = torch.randperm(num_pages, generator=g, device=device).to(torch.int32)
        width = max(1, max(need)) + (0 if tight else 2)
        self.pages = torch.full((len(past), width), -1, dtype=torch.int32, device=device)
        self.k = torch.full((num_pages, Hkv, P, 128), filler, dtype=torch.float16, device=device)
        self.v = self.k.clone()
        at = 0
        for b, c in enumerate(need):
            self.pages[b, :c] = ids[at:at + c]
            at += c
            total = self.past[b] + self.new[b]
            for pool in (self.k, self.v):
                rows = torch.randn((c * P, Hkv, 128), generator=g, device=device, dtype=torch.float16)
                rows[total:] = filler
                if window:
                    rows[:max(0, past[b] + 1 - window)] = filler  # below every new row's window
                pool[self.pages[b, :c].long()] = rows.view(c, P, Hkv, 128).transpose(1, 2)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1] + spare_rows
        self.q_starts = torch.tensor(starts, dtype=torch.int32, device=device)
        self.past_lens = torch.tensor(self.past, dtype=torch.int32, device=device)
        self.q = torch.randn((self.tokens, Hq, 128), generator=g, device=device, dtype=torch.float16)
        self.gate = 2 * torch.randn((self.tokens, Hq), generator=g, device=device)
        self.rows = starts[-1]
        self.window = window
        self.keys = max(a + n for a, n in zip(past, new))

    def check(self, be, gate=False, out_dtype=torch.float16, scale=0.0, what=""):
        pool = be.kv_pool(self.k, self.v)
        table = be.page_table(self.pages, self.past_lens, validate_on_host=False)
        out = torch.full(self.q.shape, 7.0, dtype=out_dtype, device=self.q.device)
        got = be.gqa_attention_ragged(self.q, pool, table, self.q_starts, sliding_window=self.window,
                                      gate=self.gate if gate else None, scale=scale, out=out)
        be.device_flush()
        want, size = attention_reference(self.q, self.k, self.v, self.pages, self.past, self.new, self.window,
                                         self.gate if gate else None, scale or None)
        assert_attention_close(got[:self.rows], want[:self.rows], size[:self.rows], self.keys, what)
        assert (got[self.rows:] == 7).all(), f"{what}: rows behind the last sequence were written"
        return got
