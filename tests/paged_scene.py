"""A paged cache with a batch over it, made from a seed, and what the definitions say of it in float64. Test scaffolding."""

from __future__ import annotations

import ctypes

import ml_dtypes
import numpy as np

BF16 = np.dtype(ml_dtypes.bfloat16)
F16 = np.dtype(np.float16)
NAMES = {BF16: "bfloat16", F16: "float16"}
HALF_STEP = {BF16: 2.0**-8, F16: 2.0**-11}  # a rounding to nearest is off by at most this, relative to the value
NOWHERE = 0x3FFFFFFF  # a page number that no cache has


def poison(dtype, shape) -> np.ndarray:
    """NaN everywhere."""
    return np.full(shape, 0x7FFF, dtype=np.uint16).view(dtype)


class Scene:
    """Sequences of (new tokens, keys) over pages in random order. Empty slots, pages that nobody uses, results and table
    entries past a sequence's pages hold NaN and page numbers that no cache has: whatever reads or follows one shows."""

    def __init__(self, seqs, *, dtype=BF16, heads=4, kv_heads=2, hd=64, hd_v=None, page_size=16, order="token", prefix=0, seed=0, mul=1.0,
                 spare_pages=2, spare_tokens=0, max_t_q=None, max_pages=None, row_room=0):
        rng = np.random.default_rng(seed)
        self.seqs, self.dtype, self.heads, self.kv_heads, self.hd, self.hd_v = list(seqs), dtype, heads, kv_heads, hd, hd_v or hd
        self.page_size, self.order, self.prefix = page_size, order, prefix
        self.new, self.keys = [n for n, _ in seqs], [k for _, k in seqs]
        self.start = np.cumsum([0, *self.new])
        self.tokens = int(self.start[-1]) + spare_tokens
        self.max_t_q = max_t_q or max([1, *self.new])
        used = [-(-k // page_size) for k in self.keys]
        self.max_pages = max_pages or max([1, *used])
        prefix_pages = -(-prefix // page_size)
        self.pages = sum(used) + prefix_pages + spare_pages
        free = rng.permutation(self.pages)
        self.prefix_table = free[:prefix_pages].astype(np.int32)
        self.table = np.full((max(1, len(seqs)), self.max_pages), NOWHERE, dtype=np.int32)
        at = prefix_pages
        for b, n in enumerate(used):
            self.table[b, :n] = free[at : at + n]
            at += n

        def normal(*shape):
            return rng.standard_normal(shape).astype(np.float32).astype(dtype)

        # every key there is, by sequence, and the prefix's
        self.k = [normal(k, kv_heads, self.hd) for k in self.keys]
        self.v = [normal(k, kv_heads, self.hd_v) for k in self.keys]
        self.prefix_k, self.prefix_v = normal(prefix, kv_heads, self.hd), normal(prefix, kv_heads, self.hd_v)
        self.row_room = row_room  # columns that lie between one row of q or out and the next
        self.q = (rng.standard_normal((self.tokens, heads, self.hd)) * mul).astype(np.float32).astype(dtype)

    # ---- the cache as it lies in memory: "token" (page, slot, head, column), "head" (page, head, slot, column), "roomy" as "token" with room
    # behind every head's columns, "paired" as "token" with as much again between pages (where K and V share a buffer)
    def _in_memory(self, width):
        p, s, h = self.pages, self.page_size, self.kv_heads
        return {"token": (p, s, h, width), "head": (p, h, s, width), "roomy": (p, s, h, width + 8), "paired": (p, 2 * s, h, width)}[self.order]

    def strides(self, width):
        s, h = self.page_size, self.kv_heads
        return {"token": (s * h * width, width, h * width), "head": (s * h * width, s * width, width), "roomy": (s * h * (width + 8), width + 8, h * (width + 8)),
                "paired": (2 * s * h * width, width, h * width)}[self.order]

    def by_slot(self, memory):
        if self.order == "head":
            return memory.transpose(0, 2, 1, 3)
        return memory[..., :-8] if self.order == "roomy" else memory

    def _fill(self, width, of_sequence, of_prefix, keep):
        memory = poison(self.dtype, self._in_memory(width))
        seen = self.by_slot(memory)
        for b, rows in enumerate(of_sequence):
            for j in range(keep(b)):
                seen[self.table[b, j // self.page_size], j % self.page_size] = rows[j]
        for j in range(self.prefix):
            seen[self.prefix_table[j // self.page_size], j % self.page_size] = of_prefix[j]
        return memory

    def filled(self, with_new=True):
        keep = (lambda b: self.keys[b]) if with_new else (lambda b: max(0, self.keys[b] - self.new[b]))
        return self._fill(self.hd, self.k, self.prefix_k, keep), self._fill(self.hd_v, self.v, self.prefix_v, keep)

    # ---- on the device
    def upload(self, with_new=True, first_position=None, table=None, q_start=None, kv_lens=None):
        from limn_b200 import runtime
        from limn_b200.paged import PagedBatch, PagedCache

        k, v = self.filled(with_new)
        self.k_dev, self.v_dev = runtime.upload(k), runtime.upload(v)
        self.errors = runtime.upload(np.zeros(1, np.uint32))
        self.table_dev = runtime.upload(self.table if table is None else np.asarray(table, np.int32))
        self.q_start_dev = runtime.upload(np.asarray(self.start if q_start is None else q_start, np.int32))
        self.kv_lens_dev = runtime.upload(np.asarray([*self.keys, 0] if kv_lens is None else kv_lens, np.int32))
        self.prefix_dev = runtime.upload(np.append(self.prefix_table, np.int32(NOWHERE)))
        cache = PagedCache(self.k_dev, self.v_dev, dtype=NAMES[self.dtype], pages=self.pages, page_size=self.page_size, kv_heads=self.kv_heads,
                           hd=self.hd, hd_v=self.hd_v, k_strides=self.strides(self.hd), v_strides=self.strides(self.hd_v))
        self.step = PagedBatch(cache, heads=self.heads, batch=len(self.seqs), tokens=self.tokens, max_t_q=self.max_t_q, page_table=self.table_dev,
                               max_pages=self.max_pages, q_start=self.q_start_dev, kv_lens=self.kv_lens_dev, errors=self.errors,
                               first_position=self.prefix if first_position is None else first_position, max_prefix=max(1, self.prefix))
        return self

    def error_bits(self) -> int:
        from limn_b200 import runtime

        return int(runtime.download(self.errors, np.uint32, (1,))[0])

    def attend(self, *, causal=True, scale=None, stream=None):
        """O and L as downloaded; their memory held NaN before."""
        from limn_b200 import runtime

        room = self.row_room
        q = poison(self.dtype, (self.tokens, self.heads, self.hd + room))
        q[..., : self.hd] = self.q
        q_dev = runtime.upload(q)
        out = runtime.upload(poison(self.dtype, (self.tokens, self.heads, self.hd_v + room)))
        lse = runtime.upload(np.full((self.tokens, self.heads), np.nan, np.float32))
        runtime.synchronize()
        more = {"q_strides": (self.heads * (self.hd + room), self.hd + room), "out_strides": (self.heads * (self.hd_v + room), self.hd_v + room),
                "causal": causal, "scale": scale, "stream": stream}
        if self.prefix:
            self.step.attention_with_prefix(q_dev, out, lse, prefix_table=self.prefix_dev, prefix_len=self.prefix, **more)
        else:
            self.step.attention(q_dev, out, lse, **more)
        runtime.synchronize()
        whole = runtime.download(out, np.uint16, (self.tokens, self.heads, self.hd_v + room)).view(self.dtype)
        assert (whole[..., self.hd_v :].view(np.uint16) == 0x7FFF).all(), "the room between rows was written"
        return whole[..., : self.hd_v], runtime.download(lse, np.float32, (self.tokens, self.heads))

    # ---- what the definitions say
    def expected(self, *, causal=True, scale=None):
        """O, L and A = sum p |v| / l in float64, and which tokens have a result."""
        scale = self.hd**-0.5 if scale is None else scale
        group = self.heads // self.kv_heads
        out = np.full((self.tokens, self.heads, self.hd_v), np.nan)
        size, lse = out.copy(), np.full((self.tokens, self.heads), np.nan)
        for b, (n, length) in enumerate(self.seqs):
            if n == 0:
                continue
            rows = slice(self.start[b], self.start[b] + n)
            k = np.concatenate([self.prefix_k, self.k[b]]).astype(np.float64)
            v = np.concatenate([self.prefix_v, self.v[b]]).astype(np.float64)
            j = np.arange(self.prefix + length) - self.prefix
            seen = (j[None] <= np.maximum(-1, length - n + np.arange(n))[:, None]) if causal else np.ones((n, len(j)), bool)
            for h in range(self.heads):
                s = self.q[rows, h].astype(np.float64) @ k[:, h // group].T * scale
                s[~seen] = -np.inf
                with np.errstate(invalid="ignore", divide="ignore"):
                    top = s.max(-1, initial=-np.inf, keepdims=True)
                    p = np.exp(s - np.where(np.isinf(top), 0.0, top))
                    total = p.sum(-1, keepdims=True)
                    p /= total
                    out[rows, h], size[rows, h] = p @ v[:, h // group], p @ np.abs(v[:, h // group])
                    lse[rows, h] = (top + np.log(total))[:, 0]
        return out, lse, size

    def check(self, *, causal=True, scale=None, stream=None):
        """Run and compare. O is off by its own rounding (half a step of |O|), by the rounding of the weights (half a step of
        A = sum p |v| / l) and by float32: a score of at most 128 products is off by less than 2^-14 at the sizes used here (136
        roundings of 2^-24 of sum |q k| scale < 30), and so is the weight that comes of it, in numerator and denominator:
        2^-13 A. L is off by the score's 2^-14 and by its own float32 roundings, counted as 2^-13."""
        have_o, have_l = self.attend(causal=causal, scale=scale, stream=stream)
        want_o, want_l, size = self.expected(causal=causal, scale=scale)
        self.compare(have_o, have_l, want_o, want_l, size)
        assert self.error_bits() == 0
        return have_o, have_l

    def compare(self, have_o, have_l, want_o, want_l, size):
        rows = int(self.start[-1])
        assert (have_o[rows:].view(np.uint16) == 0x7FFF).all(), "rows behind the last sequence were written"
        assert np.isnan(have_l[rows:]).all()
        have_o, have_l, want_o, want_l, size = (x[:rows] for x in (have_o, have_l, want_o, want_l, size))
        blind = np.isinf(want_l)  # rows that see no key
        assert np.array_equal(have_l == -np.inf, blind), "L = -inf in the wrong rows"
        assert np.isnan(have_o[blind].astype(np.float32)).all(), "a row that sees no key is NaN"
        seen = ~blind
        half = HALF_STEP[self.dtype]
        bound = half * np.abs(want_o[seen]) * (1 + half) + (half + 2.0**-13) * size[seen] + 2.0**-24
        off = np.abs(have_o[seen].astype(np.float64) - want_o[seen])
        assert np.isfinite(have_o[seen].astype(np.float32)).all(), "a value that is not finite"
        assert (off <= bound).all(), f"O off by {off.max():.3e}, {(off / bound).max():.2f} of what is allowed"
        off = np.abs(have_l[seen] - want_l[seen])
        assert (off <= 2.0**-13 + 2.0**-23 * np.abs(want_l[seen])).all(), f"L off by {off.max():.3e}"


def strides_of(*values):
    return (ctypes.c_longlong * len(values))(*values)
