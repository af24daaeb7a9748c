"""Plain 64-bit forms of the streaming operators, for their tests."""

import math

import numpy as np
import torch

D = 128
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # largest relative rounding error


def visible(lq, lk, window, sinks, chunk, device="cpu"):
    """bool [lq, lk]: which keys each of the last lq of lk tokens sees."""
    p = torch.arange(lk - lq, lk, device=device)[:, None]
    j = torch.arange(lk, device=device)[None]
    last = p
    if chunk > 1:
        last = torch.where(p < sinks, sinks - 1, sinks + ((p - sinks) // chunk + 1) * chunk - 1)
    see = (p >= 0) & (j <= last)
    if window is not None:
        see &= (last - j < window) | (j < sinks)
    return see


def attend(q, k, v, see, scale=None):
    """(out, spread) [lq, Hq, 128] in fp64: softmax(scale q k^T) v over `see`, and the same of |v|, what
    rounding errors of the weights are relative to.  Unseen keys take no part, whatever they hold."""
    lq, hq, _ = q.shape
    group = hq // k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(lq, hq, D, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    used = see.any(0)
    k, v, see = k[used].double(), v[used].double(), see[:, used]
    for h in range(hq):
        w = (q[:, h].double() @ k[:, h // group].T) * scale
        w = w.masked_fill(~see, -math.inf)
        top = w.amax(-1, keepdim=True) if w.shape[1] else w.new_zeros(lq, 1)
        w = torch.exp(w - top.clamp_min(-1e300))
        w = w.masked_fill(~see, 0.0)
        total = w.sum(-1, keepdim=True)
        w = w / total.clamp_min(1e-300)
        # an unseen row may hold anything: it must not meet the weight 0
        out[:, h] = w @ v[:, h // group]
        spread[:, h] = w @ v[:, h // group].abs()
    return out, spread


def tolerance(out, spread, dtype, keys, vmax):
    """|error| allowed: the output's rounding, the rounding of each weight to the 16-bit type of the V
    product (fp16 weights below 2^-14 have an absolute step of 2^-24), and 2e-4 for fp32 scores of
    magnitude up to 60 (2^-24 * 60 * sqrt(128) * ln-scale) with the exponential's relative error (< 1e-4)."""
    u = UNIT[dtype]
    tiny = keys * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    return u * out.abs() + (u + 2e-4) * spread * (1 + u) + tiny + 1e-30


def assert_close(got, ref, spread, keys, vmax, what=""):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got.double() - ref).abs()
    tol = tolerance(ref, spread, got.dtype, keys, vmax)
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.2f} x tolerance"


class HostCache:
    """The page work of a paged cache, step by step on the host (numpy tables, torch pools)."""

    def __init__(self, cache):
        self.page = cache.k.shape[3]
        self.k, self.v = cache.k.clone(), cache.v.clone()
        self.table, self.lens, self.refs = (x.cpu().numpy().copy() for x in (cache.table, cache.lens, cache.refs))
        self.k_scale, self.v_scale = cache.k_scale, cache.v_scale

    def pages_of(self, n):
        return -(-int(n) // self.page)

    def extend(self, slots, counts):
        shared = self.refs.copy()
        given, dropped = [], []
        for s, n in zip(slots, counts):
            last = self.table[s, self.lens[s] // self.page] if self.lens[s] % self.page else -1
            if n and last >= 0 and shared[last] > 1:
                new = int(np.flatnonzero(self.refs == 0)[0])
                self.refs[new] = 1
                dropped.append(last)
                self.table[s, self.lens[s] // self.page] = new
                part = int(self.lens[s] % self.page)
                for pool in (self.k, self.v):
                    raw = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)
                    raw[:, new, :, :part] = raw[:, int(last), :, :part].clone()
            for col in range(self.pages_of(self.lens[s]), self.pages_of(self.lens[s] + n)):
                new = int(np.flatnonzero(self.refs == 0)[0])
                self.refs[new] = 1
                self.table[s, col] = new
            self.lens[s] += n
        for p in dropped:
            self.refs[p] -= 1

    def write(self, slots, counts, k, v, layer=0):
        at = 0
        for s, n in zip(slots, counts):
            for i in range(n):
                pos = int(self.lens[s]) - n + i
                p, o = int(self.table[s, pos // self.page]), pos % self.page
                for pool, x, scale in ((self.k, k, self.k_scale), (self.v, v, self.v_scale)):
                    row = x[at + i]
                    if scale is not None:
                        row = (row.float() / scale[layer][:, None]).clamp(-448, 448)
                    raw = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)
                    raw[layer, p, :, o] = row.to(pool.dtype).view(raw.dtype)
            at += n

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            self.table[b], self.lens[b] = self.table[a], self.lens[a]
            for p in self.table[b][self.table[b] >= 0]:
                self.refs[p] += 1

    def truncate(self, slots, keep):
        for s, n in zip(slots, keep):
            for col in range(self.pages_of(n), self.pages_of(self.lens[s])):
                self.refs[self.table[s, col]] -= 1
                self.table[s, col] = -1
            self.lens[s] = n

    def compact(self):
        used = np.flatnonzero(self.refs)
        n = used.size
        for new, old in zip(np.flatnonzero(self.refs[:n] == 0), used[used >= n]):
            for pool in (self.k, self.v):
                raw = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)
                raw[:, int(new)] = raw[:, int(old)].clone()
            self.refs[new], self.refs[old] = self.refs[old], 0
            self.table[self.table == old] = new

    def assert_equal(self, cache, what=""):
        for name in ("table", "lens", "refs"):
            got = getattr(cache, name).cpu().numpy()
            assert np.array_equal(got, getattr(self, name)), f"{what}: {name} differs"
        for name in ("k", "v"):
            got, want = getattr(cache, name), getattr(self, name)
            raw = torch.uint8 if got.element_size() == 1 else torch.int16
            assert torch.equal(got.view(raw), want.view(raw)), f"{what}: {name} differs"

    def rows(self, slot, layer=0):
        """K, V [tokens, kv heads, 128] in fp64 of a sequence."""
        n = int(self.lens[slot])
        out = []
        for pool, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            pages = self.table[slot, : self.pages_of(n)].tolist()
            x = [pool[layer, p].double().transpose(0, 1) for p in pages]
            x = torch.cat(x)[:n] if x else torch.zeros(0, pool.shape[2], D, dtype=torch.float64, device=pool.device)
            out.append(x if scale is None else x * scale[layer].double()[:, None])
        return out
