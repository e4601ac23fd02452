"""Positions, cache and attention of a model's attention layers for several sequences, over the library's entry points.

``rope_freq`` makes the frequencies dr_rope takes, scaled for contexts longer than the trained one.  ``KvCache`` owns the pages
of all layers and says which sequence holds which (host side); ``KvCache.step`` makes a ``Batch`` of new rows, which
``rope``, ``append``, ``attend`` and ``read`` of every layer then share.  Kernels and copies go to torch's current stream of the
cache's device; there is no host round trip in them, so they can be captured after a first call on the stream.
"""
from __future__ import annotations

import math

import dramamoe

BLOCK = dramamoe.header_define("DR_KV8_BLOCK")
HALF, PAIRS = dramamoe.header_define("DR_ROPE_HALF"), dramamoe.header_define("DR_ROPE_PAIRS")


def rope_freq(rot: int, theta: float = 10000.0, scaling: str | None = None, factor: float = 1.0, trained: int = 4096,
              fast: float = 32.0, slow: float = 1.0, device=None):
    """(freq f32 [rot / 2], mscale) of dr_rope for ``rot`` rotated elements.

    theta ** (-2 j / rot) and 1, or for a context ``factor`` times as long as the ``trained`` one:
      "linear"  every frequency over factor (positions drawn together);
      "base"    theta * factor ** (rot / (rot - 2)), so that the slowest frequency is the one drawn out by factor;
      "yarn"    a frequency that turns more than ``fast`` times within the trained length stays, one that turns less than ``slow`` times is
                divided by factor, those between are mixed linearly in j; mscale 0.1 ln(factor) + 1."""
    import torch

    if rot < 0 or rot % 2:
        raise ValueError(f"rot {rot}: even, not negative")
    if scaling not in (None, "linear", "base", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not factor >= 1 or not theta > 1:
        raise ValueError("factor at least 1, theta above 1")
    if scaling == "base" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    j = torch.arange(rot // 2, dtype=torch.float64)
    f = theta ** (-2 * j / max(rot, 1))
    mscale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        # the (real) j at which a frequency turns `turns` times within the trained length
        at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
        keep = 1 - ((j - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f, mscale = f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return f.float().to(device or "cpu"), mscale


def _check_rows(t, rows, width, dtypes, device, what):
    if t.device != device or t.dtype not in dtypes or t.dim() != 2 or t.shape[0] < rows or t.shape[1] != width or t.stride(1) != 1:
        raise ValueError(f"{what}: {tuple(t.shape)} {t.dtype} on {t.device}, expected [{rows}, {width}] of {dtypes} on {device}")


class Batch:
    """New rows of a call: sequence i has rows start[i] .. start[i + 1] - 1, len[i] tokens with them, row r the position pos[r]."""

    def __init__(self, rows, lens, device):
        import torch

        start = [0]
        for n in rows:
            start.append(start[-1] + n)
        self.rows, self.total, self.max_rows, self.max_len = list(rows), start[-1], max(rows, default=0), max(lens, default=0)
        self.pos = torch.tensor([m - n + r for n, m in zip(rows, lens) for r in range(n)], dtype=torch.int32, device=device)
        self.start = torch.tensor(start, dtype=torch.int32, device=device)
        self.len = torch.tensor(list(lens), dtype=torch.int32, device=device)
        self.seqs, self.device = len(start) - 1, self.start.device


class KvCache:
    """k and v in 8 bits of ``layers`` layers for up to ``seqs`` sequences of up to ``max_len`` tokens, in ``pages`` pages of 64 tokens a layer that
    the sequences share.  hq queries and hkv cached heads of d elements (a multiple of 16 up to 256)."""

    def __init__(self, layers: int, pages: int, seqs: int, max_len: int, hq: int, hkv: int, d: int, device="cuda"):
        import torch

        if layers < 1 or pages < 1 or seqs < 1 or max_len < 1 or hkv < 1 or hq < 1 or hq % hkv or hq > 1024 or d % 16 or not 16 <= d <= 256:
            raise ValueError(f"no cache of {layers} layers, {pages} pages, {seqs} sequences of {max_len}, heads {hq} / {hkv} of {d}")
        self.layers, self.pages, self.seqs, self.hq, self.hkv, self.d = layers, pages, seqs, hq, hkv, d
        self.maxp = (max_len + BLOCK - 1) // BLOCK
        self.max_len = max_len
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        z = lambda *s, dt=torch.uint8: torch.zeros(s, dtype=dt, device=self.device)
        self.kq, self.vq = z(layers, pages, hkv, d // 16, BLOCK, 16), z(layers, pages, hkv, d, BLOCK)
        self.ks, self.vs = z(layers, pages, hkv, dt=torch.float32), z(layers, pages, hkv, dt=torch.float32)
        self.table = torch.full((seqs, self.maxp), -1, dtype=torch.int32, device=self.device)
        self.lens = [0] * seqs
        self.held = [[] for _ in range(seqs)]  # pages of each sequence, in order
        self.free_pages = list(range(pages - 1, -1, -1))
        self._ws = {}   # stream handle -> workspace of attend
        self._old = []  # smaller ones that a captured call may still use
        self.lib = dramamoe.lib()

    # ---- which sequence holds what (host side) ----

    def step(self, rows) -> Batch:
        """rows[i] new tokens for sequence i: takes the pages they need and counts them in.  Nothing changes where that is not possible."""
        import torch

        rows = [int(n) for n in rows]
        if len(rows) != self.seqs or any(n < 0 for n in rows):
            raise ValueError(f"a number of rows for each of the {self.seqs} sequences")
        need = []
        for i, n in enumerate(rows):
            if self.lens[i] + n > self.max_len:
                raise ValueError(f"sequence {i}: {self.lens[i] + n} tokens of at most {self.max_len}")
            need.append((self.lens[i] + n + BLOCK - 1) // BLOCK - len(self.held[i]))
        if sum(need) > len(self.free_pages):
            raise MemoryError(f"{sum(need)} pages needed, {len(self.free_pages)} free")
        # what can fail comes before what is counted
        lens = [m + n for m, n in zip(self.lens, rows)]
        batch = Batch(rows, lens, self.device)
        new = self.free_pages[len(self.free_pages) - sum(need):][::-1]
        at = [i * self.maxp + len(self.held[i]) + k for i in range(self.seqs) for k in range(need[i])]
        if at:
            self.table.view(-1)[torch.tensor(at, device=self.device)] = torch.tensor(new, dtype=torch.int32, device=self.device)
            del self.free_pages[-len(new):]
        pages = iter(new)
        for i, k in enumerate(need):
            self.held[i] += [next(pages) for _ in range(k)]
        self.lens = lens
        return batch

    def truncate(self, seq: int, length: int) -> None:
        """Keeps the first ``length`` tokens of a sequence and gives back the pages behind them (0: all; drafted tokens that were refused).
        Pages given back may be taken by the next ``step``: calls over them must have been issued to the same stream.  A block that is kept in
        part keeps what the tokens taken back made of it: a scale that they made grow, with the kept tokens' integers rounded to it, and NaN where
        one of them was no number.  Where that matters, drafts are kept from the cache until they are accepted."""
        if not 0 <= length <= self.lens[seq]:
            raise ValueError(f"sequence {seq} has {self.lens[seq]} tokens, not {length}")
        keep = (length + BLOCK - 1) // BLOCK
        while len(self.held[seq]) > keep:
            self.free_pages.append(self.held[seq].pop())
        self.table[seq, keep:] = -1
        self.lens[seq] = length

    # ---- what runs on the device ----

    def _check(self, t, rows, width, dtypes, what):
        _check_rows(t, rows, width, dtypes, self.device, what)

    def _check_batch(self, batch):
        # the kernels read start and len of every sequence of the cache
        if batch.seqs != self.seqs or batch.device != self.device:
            raise ValueError(f"a batch of {batch.seqs} sequences on {batch.device}, expected {self.seqs} on {self.device}")

    def _cache(self, layer):
        P = dramamoe.ptr
        return (P(self.table), self.maxp, P(self.kq[layer]), P(self.ks[layer]), P(self.vq[layer]), P(self.vs[layer]), self.pages)

    def _on_device(self):
        import torch

        return torch.cuda.device(self.device)

    def append(self, layer: int, k, v, batch: Batch) -> None:
        """k and v (f32, or both bf16) [batch.total, hkv * d] become the new tokens of ``layer``."""
        import torch

        n = self.hkv * self.d
        self._check_batch(batch)
        for t, what in ((k, "k"), (v, "v")):
            self._check(t, batch.total, n, (torch.float32, torch.bfloat16), what)
        if k.dtype != v.dtype:
            raise ValueError("k and v of one type")
        f = self.lib.dr_kv8_append_bf16 if k.dtype == torch.bfloat16 else self.lib.dr_kv8_append
        with self._on_device():
            f(k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), dramamoe.ptr(batch.start), dramamoe.ptr(batch.len), *self._cache(layer), batch.total,
              self.seqs, self.hkv, self.d, dramamoe.stream_ptr())

    def read(self, layer: int, batch: Batch):
        """(k, v) f32 [batch.total, hkv * d]: the values that the cache holds for the batch's rows."""
        import torch

        n, P = self.hkv * self.d, dramamoe.ptr
        self._check_batch(batch)
        with self._on_device():
            k, v = (torch.empty(batch.total, n, device=self.device) for _ in range(2))
            self.lib.dr_kv8_read(P(batch.start), P(batch.len), *self._cache(layer), P(k), n, P(v), n, batch.total, self.seqs, self.hkv, self.d,
                                 dramamoe.stream_ptr())
        return k, v

    def attend(self, layer: int, q, batch: Batch, scale: float | None = None, gate=None, out=None, max_len: int | None = None,
               gate_stride: int | None = None):
        """Attention of the batch's rows (their tokens appended before) over ``layer``: q bf16 [batch.total, hq * d], gate None or f32 of
        that shape, -> bf16 of that shape (``out``, which may be q).  scale: d ** -0.5.  gate_stride: elements from a head's gate to the next
        one's, d where the heads' gates lie side by side; 2 * d where each lies beside its query: gate is then the projection's [batch.total, (2 hq - 1) d]
        from the first gate on.  max_len: a captured call that is replayed while the
        sequences grow takes their final length here.  Captured calls keep the stream's workspace: graphs that may run at the same
        time are captured on streams of their own."""
        import torch

        n, P = self.hq * self.d, dramamoe.ptr
        self._check_batch(batch)
        self._check(q, batch.total, n, (torch.bfloat16,), "q")
        if gate is not None:
            hsg = self.d if gate_stride is None else gate_stride
            self._check(gate, batch.total, (self.hq - 1) * hsg + self.d, (torch.float32,), "gate")
        if out is not None:
            self._check(out, batch.total, n, (torch.bfloat16,), "out")
        longest = batch.max_len if max_len is None else max_len
        with self._on_device():
            if out is None:
                out = torch.empty(batch.total, n, dtype=torch.bfloat16, device=self.device)
            st = dramamoe.stream_ptr()
            size = self.lib.dr_attn_kv8_ws(batch.total, self.seqs, batch.max_rows, longest, self.hq, self.hkv, self.d)
            if size == 0:
                raise ValueError("no attention kernel for this shape")
            ws = self._ws.get(st)
            if ws is None or ws.numel() < size:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("call attend once on this stream, with as many rows and tokens, before capturing it")
                if ws is not None:
                    # at least doubled, so that all that were outgrown together are smaller than the one in use
                    self._old.append(ws)
                    size = max(size, 2 * ws.numel())
                ws = self._ws[st] = torch.empty(size, dtype=torch.uint8, device=self.device)
            self.lib.dr_attn_kv8(q.data_ptr(), q.stride(0), P(batch.start), P(batch.len), *self._cache(layer), self.d ** -0.5 if scale is None else scale,
                                 None if gate is None else gate.data_ptr(), 0 if gate is None else gate.stride(0), 0 if gate is None else hsg, P(ws), out.data_ptr(),
                                 out.stride(0), batch.total, self.seqs, batch.max_rows, longest, self.hq, self.hkv, self.d, st)
        return out


def rope(x, heads: int, d: int, pos, freq, mscale: float = 1.0, layout: int = HALF, nw=None, eps: float = 1e-6, head_stride: int | None = None,
         f32: bool = False, out=None):
    """dr_rope on x (f32 or bf16, rows of ``heads`` heads head_stride or d elements apart): bf16 [rows, heads * d], f32 where ``f32``, or into ``out`` (f32
    or bf16 of that shape; x itself where its heads lie side by side and the types are the same).  nw None, or f32 [d] or [heads, d]; freq f32 [rot / 2], of which the first rot elements of a head are turned."""
    import torch

    P, hs, n = dramamoe.ptr, head_stride or d, heads * d
    if x.dtype not in (torch.float32, torch.bfloat16) or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < (heads - 1) * hs + d:
        raise ValueError(f"x: {tuple(x.shape)} {x.dtype}")
    if pos.dtype != torch.int32 or pos.numel() < x.shape[0] or freq.dtype != torch.float32 or 2 * freq.numel() > d:
        raise ValueError("pos i32 [rows], freq f32 [rot / 2] with rot <= d")
    if nw is not None and (nw.dtype != torch.float32 or nw.numel() not in (d, heads * d)):
        raise ValueError("nw f32 [d] or [heads, d]")
    if any(t is not None and t.device != x.device for t in (pos, freq, nw)):
        raise ValueError("pos, freq and nw on the device of x")
    if out is not None:
        _check_rows(out, x.shape[0], n, (torch.float32, torch.bfloat16), x.device, "out")
        f32 = out.dtype == torch.float32
    lib = dramamoe.lib()
    f = lib.dr_rope_bf16 if x.dtype == torch.bfloat16 else lib.dr_rope
    with torch.cuda.device(x.device):
        if out is None:
            out = torch.empty(x.shape[0], n, dtype=torch.float32 if f32 else torch.bfloat16, device=x.device)
        y, ldy = out.data_ptr(), out.stride(0)
        f(x.data_ptr(), x.stride(0), hs, P(nw), 0 if nw is None or nw.numel() == d else d, eps, P(pos), P(freq), mscale, layout,
          y if f32 else None, ldy, None if f32 else y, ldy, x.shape[0], heads, d, 2 * freq.numel(), dramamoe.stream_ptr())
    return out
