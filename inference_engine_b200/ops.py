"""Decoder ops in the model's own precision (bf16 or fp32), over libb200dec.so (include/b200dec.h).

They stand beside `kernels` (the int8-cache attention path with the reference's signatures) and cover what a decoder of
another design needs: a paged KV cache of unquantised rows whose key and value sizes are free of one another, partial
rotary positions with frequency scaling, unit-norm heads, a 32-bit residual stream normed after the sum, and a mixture of
experts.  Every constant of a design is an argument.  As in `kernels` there is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib
from . import kernels as K

MAX_TENSOR_CORE_DIM = 128  # head sizes up to this run on the tensor-core attention kernels (bf16)


def _lib_dec():
    return _lib.load_decoder()


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _elem(dtype: torch.dtype) -> int:
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"decoder ops run in bfloat16 or float32, not {dtype}")
    return 2 if dtype == torch.bfloat16 else 4


def _round8(n: int) -> int:
    return (n + 7) // 8 * 8


# ----------------------------------------------------------------------------- the paged cache of unquantised rows
@dataclass
class PagedKV:
    """One layer's keys and values, rows padded to 8 channels (the padding stays zero)."""

    k: torch.Tensor  # [num_pages, kv_heads, page_size, round8(k_dim)]
    v: torch.Tensor  # [num_pages, kv_heads, page_size, round8(v_dim)]
    k_dim: int
    v_dim: int

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def struct(self) -> _lib.DecCache:
        k, v = self.k, self.v
        return _lib.DecCache(k.data_ptr(), v.data_ptr(), k.shape[0], k.shape[1], k.shape[2], self.k_dim, self.v_dim, k.shape[3],
                             v.shape[3], k.element_size())


def make_paged_kv(num_pages: int, kv_heads: int, page_size: int, k_dim: int, v_dim: int, dtype, device) -> PagedKV:
    def z(d):
        return torch.zeros(num_pages, kv_heads, page_size, _round8(d), dtype=dtype, device=device)

    return PagedKV(z(k_dim), z(v_dim), k_dim, v_dim)


@dataclass
class Rows:
    """Which (entry, position) each packed row of a step is.  seq_ids / positions None: pure decode, row = entry at
    position cached_lens[row], rows from num_decoding on idle.  cu_seqlens and tile_start (the entries' and tiles' first rows) are what recurrent layers
    and the tensor cores' attention go by, whose rows lie entry after entry at consecutive positions; 32-bit attention goes by seq_ids and positions."""

    num_rows: int
    cached_lens: torch.Tensor
    num_decoding: torch.Tensor
    block_table: torch.Tensor  # int32 [entries, max_pages]
    seq_ids: torch.Tensor | None = None
    positions: torch.Tensor | None = None
    cu_seqlens: torch.Tensor | None = None
    tile_start: torch.Tensor | None = None
    block_m: int = 128
    slots: torch.Tensor | None = None  # int32 [entries]: state slots of recurrent layers, -1 = passed over

    def struct(self) -> _lib.DecRows:
        return _lib.DecRows(_ptr(self.seq_ids), _ptr(self.positions), K._i32(self.cached_lens), K._i32(self.num_decoding),
                            self.num_rows)

    def entries(self) -> _lib.Entries:
        return _lib.Entries(_ptr(self.cu_seqlens), K._i32(self.cached_lens), K._i32(self.num_decoding), K._i32(self.slots),
                            _ptr(self.seq_ids), _ptr(self.positions), self.cached_lens.shape[0], self.num_rows)


# ----------------------------------------------------------------------------- rotary positions
@dataclass(frozen=True)
class Rotary:
    """Rotation of the first `dims` channels of a head, channel i paired with i + dims / 2 (rope_write) or 2i with 2i + 1
    (norm_rope_write).  With `scaling` (factor,
    original, fast, slow) the frequencies are stretched as YaRN does (Peng et al., "YaRN: Efficient Context Window
    Extension of Large Language Models"): components that turn more than `fast` times within the original context
    keep their frequency, those that turn less than `slow` times are divided by `factor`, a linear ramp joins the two,
    and cos and sin are multiplied by 0.1 ln(factor) + 1."""

    dims: int
    base: float
    scaling: tuple[float, float, float, float] | None = None  # factor, original, fast, slow
    stretch: float = 1.0  # linear scaling: every frequency is divided by it

    def frequencies(self) -> tuple[list[float], float]:
        half = self.dims // 2
        freq = [self.base ** (-2.0 * i / self.dims) / self.stretch for i in range(half)]
        if self.scaling is None:
            return freq, 1.0
        factor, original, fast, slow = self.scaling

        def component(turns: float) -> float:
            return self.dims * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(self.base))

        lo = max(math.floor(component(fast)), 0)
        hi = min(math.ceil(component(slow)), self.dims - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(half)]
        return [f / factor * r + f * (1.0 - r) for f, r in zip(freq, ramp)], 0.1 * math.log(factor) + 1.0

    def table(self, length: int, device) -> torch.Tensor:
        """fp32 [length, dims / 2, 2]: cos and sin of every position, multiplier included (angles in 64-bit)."""
        freq, mult = self.frequencies()
        pos = torch.arange(length, dtype=torch.float64, device=device)
        a = pos[:, None] * torch.tensor(freq, dtype=torch.float64, device=device)
        return (torch.stack((a.cos(), a.sin()), dim=-1) * mult).to(torch.float32).contiguous()


# ----------------------------------------------------------------------------- row ops
@K._ranged
def embed(table: torch.Tensor, ids: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(residual rows fp32, the same rows in the model's precision; one tensor when that is fp32)."""
    K._require_cuda(table, ids)
    assert ids.dtype == torch.int32 and table.is_contiguous()
    N, W = ids.shape[0], table.shape[1]
    x = torch.empty(N, W, device=ids.device, dtype=torch.float32)
    xb = x if table.dtype == torch.float32 else torch.empty(N, W, device=ids.device, dtype=table.dtype)
    rc = _lib_dec().b200dec_embed(table.data_ptr(), _elem(table.dtype), ids.data_ptr(), x.data_ptr(), None if xb is x else xb.data_ptr(),
                                  N, W, table.shape[0], K.status_word(ids.device).data_ptr(), K._stream())
    _lib.check(rc, "embed")
    return x, xb


@K._ranged
def scaled_add_norm(x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, alpha: float, eps: float, dtype: torch.dtype,
                    index: torch.Tensor | None = None, keep: bool = True, zero: torch.Tensor | None = None):
    """y = rmsnorm(alpha * x + delta) * weight, all in 32-bit; (y fp32 written over x, y in `dtype`).  `index` int32
    [rows, top]: delta is the sum of those rows of it.  keep = False: only the copy in `dtype` is made.  `zero`: an
    int32 tensor cleared on the way."""
    K._require_cuda(x, weight)
    assert x.dtype == torch.float32 and x.is_contiguous() and weight.dtype == torch.float32
    assert delta is None or (delta.is_contiguous() and delta.dtype == dtype)
    N, W = x.shape
    xb = None
    if dtype != torch.float32 or not keep:
        xb = torch.empty(N, W, device=x.device, dtype=dtype)
    rc = _lib_dec().b200dec_scaled_add_norm(
        x.data_ptr(), _ptr(delta), _ptr(index), 1 if index is None else index.shape[1], _elem(dtype), weight.data_ptr(), float(alpha),
        float(eps), x.data_ptr() if keep else None, _ptr(xb), N, W, _ptr(zero), 0 if zero is None else zero.numel(), K._stream())
    _lib.check(rc, "scaled_add_norm")
    return x, (x if xb is None else xb)


@K._ranged
def norm_add(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, mult: float, eps: float, dtype: torch.dtype) -> torch.Tensor:
    """x += mult * rmsnorm(y) * weight in 32-bit, in place; returns the new rows in `dtype` (x itself when that is fp32)."""
    K._require_cuda(x, y, weight)
    assert x.dtype == weight.dtype == torch.float32 and x.is_contiguous() and y.is_contiguous() and y.shape == x.shape and y.dtype == dtype
    xb = x if dtype == torch.float32 else torch.empty_like(x, dtype=dtype)
    rc = _lib_dec().b200dec_norm_add(x.data_ptr(), y.data_ptr(), _elem(dtype), weight.data_ptr(), float(mult), float(eps),
                                     None if xb is x else xb.data_ptr(), x.shape[0], x.shape[1], K._stream())
    _lib.check(rc, "norm_add")
    return xb


@K._ranged
def silu_mul(gate_up: torch.Tensor, ff: int) -> torch.Tensor:
    """silu(gate) * up of rows gate [ff] | up [ff]."""
    K._require_cuda(gate_up)
    assert gate_up.stride(1) == 1 and gate_up.shape[1] >= 2 * ff
    out = torch.empty(gate_up.shape[0], ff, device=gate_up.device, dtype=gate_up.dtype)
    rc = _lib_dec().b200dec_silu_mul(gate_up.data_ptr(), gate_up.stride(0), gate_up.element_size(), out.data_ptr(), ff, gate_up.shape[0], ff,
                                     K._stream())
    _lib.check(rc, "silu_mul")
    return out


# ----------------------------------------------------------------------------- attention
@K._ranged
def rope_write(qkv: torch.Tensor, rows: Rows, cache: PagedKV, cos_sin: torch.Tensor | None, heads: int, write_kv: bool, unit_norm: bool,
               eps: float) -> torch.Tensor:
    """Rotated (and, with unit_norm, unit root-mean-square) queries [N, heads, round8(k_dim)]; keys and values of the
    rows are written to the cache unless write_kv is False (the layer then attends another layer's cache)."""
    K._require_cuda(qkv, cache.k)
    assert qkv.dtype == cache.k.dtype and qkv.stride(1) == 1
    assert qkv.shape[1] == heads * cache.k_dim + (cache.kv_heads * (cache.k_dim + cache.v_dim) if write_kv else 0)
    q = torch.empty(rows.num_rows, heads, cache.k.shape[3], device=qkv.device, dtype=qkv.dtype)
    cs, ts, rs = cache.struct(), K._table_struct(rows.block_table), rows.struct()
    rc = _lib_dec().b200dec_rope_write(
        qkv.data_ptr(), qkv.stride(0), ctypes.byref(rs), ctypes.byref(cs), ctypes.byref(ts), _ptr(cos_sin),
        0 if cos_sin is None else cos_sin.shape[0], 0 if cos_sin is None else cos_sin.shape[1], heads, int(write_kv), int(unit_norm),
        float(eps), q.data_ptr(), K.status_word(qkv.device).data_ptr(), K._stream())
    _lib.check(rc, "rope_write")
    return q


@K._ranged
def norm_rope_write(qkv: torch.Tensor, rows: Rows, cache: PagedKV, q_norm: torch.Tensor, k_norm: torch.Tensor, eps: float,
                    cos_sin: torch.Tensor | None, heads: int) -> torch.Tensor:
    """As rope_write with the RMS norm over the whole query projection and the whole key projection (weights fp32), before
    a rotation that pairs channels 2i and 2i + 1."""
    K._require_cuda(qkv, cache.k, q_norm, k_norm)
    assert qkv.dtype == cache.k.dtype and qkv.stride(1) == 1 and q_norm.dtype == k_norm.dtype == torch.float32
    assert qkv.shape[1] == heads * cache.k_dim + cache.kv_heads * (cache.k_dim + cache.v_dim)
    assert q_norm.numel() == heads * cache.k_dim and k_norm.numel() == cache.kv_heads * cache.k_dim
    q = torch.empty(rows.num_rows, heads, cache.k.shape[3], device=qkv.device, dtype=qkv.dtype)
    cs, ts, rs = cache.struct(), K._table_struct(rows.block_table), rows.struct()
    rc = _lib_dec().b200dec_norm_rope_write(
        qkv.data_ptr(), qkv.stride(0), ctypes.byref(rs), ctypes.byref(cs), ctypes.byref(ts), q_norm.data_ptr(), k_norm.data_ptr(), float(eps),
        _ptr(cos_sin), 0 if cos_sin is None else cos_sin.shape[0], 0 if cos_sin is None else cos_sin.shape[1], heads, q.data_ptr(),
        K.status_word(qkv.device).data_ptr(), K._stream())
    _lib.check(rc, "norm_rope_write")
    return q


@dataclass
class AttnOptions:
    """window: a row sees itself and the window - 1 tokens before it (0: all).  sink fp32 [heads]: exp(sink) joins the
    softmax denominator.  gate [rows, heads] in the model's precision: head outputs times sigmoid(gate).  out_scale
    multiplies the result."""

    window: int = 0
    sink: torch.Tensor | None = None
    gate: torch.Tensor | None = None
    out_scale: float = 1.0

    def struct(self, out: torch.Tensor) -> _lib.AttnOptions:
        assert self.sink is None or (self.sink.dtype == torch.float32 and self.sink.is_contiguous())
        assert self.gate is None or (self.gate.stride(1) == 1 and self.gate.dtype == out.dtype)
        return _lib.AttnOptions(self.window, _ptr(self.sink), _ptr(self.gate), 0 if self.gate is None else self.gate.stride(0),
                                self.out_scale, out.stride(0))


def _opt(opt: AttnOptions | None, out: torch.Tensor):
    """The option argument of an attention call; `out` [rows, heads, v_dim] may be a part of wider rows with options only."""
    assert out.stride(2) == 1 and out.stride(1) == out.shape[2]
    if opt is None and out.is_contiguous():
        return None
    st = (opt or AttnOptions()).struct(out)
    if out.is_contiguous():
        st.out_stride = 0
    return ctypes.byref(st)


def tensor_core_attention(cache: PagedKV) -> bool:
    return cache.k.dtype == torch.bfloat16 and max(cache.k_dim, cache.v_dim) <= MAX_TENSOR_CORE_DIM and cache.page_size % 16 == 0


@K._ranged
def attention_rows(q: torch.Tensor, cache: PagedKV, rows: Rows, scale: float, opt: AttnOptions | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of every row over the cache on the CUDA cores, 32-bit: any sizes, both precisions."""
    K._require_cuda(q, cache.k)
    if out is None:
        out = torch.empty(q.shape[0], q.shape[1], cache.v_dim, device=q.device, dtype=q.dtype)
    cs, ts, rs = cache.struct(), K._table_struct(rows.block_table), rows.struct()
    cu = rows.cu_seqlens
    if cu is not None and (cu.dtype != torch.int32 or not cu.is_contiguous() or cu.device != q.device or cu.numel() < 2):
        cu = None  # it only says how the rows are shared out
    rc = _lib_dec().b200dec_attn_rows_entries(q.data_ptr(), ctypes.byref(cs), ctypes.byref(ts), ctypes.byref(rs),
                                              _ptr(cu), 0 if cu is None else cu.numel() - 1, q.shape[1], float(scale),
                                              _opt(opt, out), out.data_ptr(), K.status_word(q.device).data_ptr(), K._stream())
    _lib.check(rc, "attention_rows")
    return out


@K._ranged
def paged_decode_attention(q: torch.Tensor, cache: PagedKV, rows: Rows, scale: float, out: torch.Tensor, zero_idle: bool,
                           opt: AttnOptions | None = None) -> None:
    """The decoding entries' rows (the first ones of q and out) on the tensor cores."""
    K._require_cuda(q, cache.k)
    lib, dev, sms = _lib_dec(), q.device, K.num_sms(q.device)
    B, heads = rows.cached_lens.shape[0], q.shape[1]
    nbytes = lib.b200dec_decode_attn_workspace(B, heads, cache.kv_heads, cache.v_dim, sms)
    ws = K.decode_workspace(dev, ("paged", B, cache.v_dim), heads, cache.kv_heads, nbytes)
    cs, ts = cache.struct(), K._table_struct(rows.block_table)
    rc = lib.b200dec_decode_attn_opt(q.data_ptr(), ctypes.byref(cs), ctypes.byref(ts), K._i32(rows.cached_lens), K._i32(rows.num_decoding),
                                     B, heads, float(scale), _opt(opt, out), out.data_ptr(), int(zero_idle), ws.data_ptr(), ws.numel(), sms,
                                     K.status_word(dev).data_ptr(), K._stream())
    _lib.check(rc, "paged_decode_attention")


@K._ranged
def paged_prefill_attention(q: torch.Tensor, cache: PagedKV, rows: Rows, scale: float, out: torch.Tensor,
                            opt: AttnOptions | None = None) -> None:
    """The prompt portions' rows on tcgen05, keys and values by page from the cache."""
    K._require_cuda(q, cache.k)
    cs, ts = cache.struct(), K._table_struct(rows.block_table)
    rc = _lib_dec().b200dec_prefill_attn_opt(
        q.data_ptr(), ctypes.byref(cs), ctypes.byref(ts), K._i32(rows.seq_ids), K._i32(rows.cu_seqlens), K._i32(rows.cached_lens),
        K._i32(rows.tile_start), rows.tile_start.shape[0], rows.block_m, rows.num_rows, q.shape[1], float(scale), _opt(opt, out),
        out.data_ptr(), K.status_word(q.device).data_ptr(), K._stream())
    _lib.check(rc, "paged_prefill_attention")


def paged_attention(q: torch.Tensor, cache: PagedKV, rows: Rows, scale: float, opt: AttnOptions | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's rows over the paged cache: [N, heads, v_dim] (written to `out` if given)."""
    if not tensor_core_attention(cache):
        return attention_rows(q, cache, rows, scale, opt, out)
    if out is None:
        out = torch.empty(q.shape[0], q.shape[1], cache.v_dim, device=q.device, dtype=q.dtype)
    if rows.seq_ids is None:
        paged_decode_attention(q, cache, rows, scale, out, True, opt)
        return out
    if not K.recording():
        paged_prefill_attention(q, cache, rows, scale, out, opt)
        paged_decode_attention(q, cache, rows, scale, out, False, opt)
        return out
    # Rows of portions and of decoding entries: neither reads what the other writes.  us with the row writes, 16 heads in bf16: 32 entries
    # beside 992 rows on 3072 100 -> 84, 8 beside 2 x 50 rows on 300 32.8 -> 18.7, five prompts of 1000 rows 34.9 -> 22.6.
    with K.Branches(_lib_dec()) as both:
        paged_prefill_attention(q, cache, rows, scale, out, opt)
        both.next()
        paged_decode_attention(q, cache, rows, scale, out, False, opt)
    return out


# ----------------------------------------------------------------------------- mixture of experts
@dataclass
class Experts:
    """Weights of one layer's experts: gate and up rows interleaved (row 2f = gate f, row 2f + 1 = up f), so that one
    product yields both inputs of an output channel side by side."""

    router: torch.Tensor  # bf16 [experts, width]
    gate_up: torch.Tensor  # [experts, 2 * ff, width]
    down: torch.Tensor  # [experts, width, ff]
    top: int
    limit: float
    slope: float
    counts: torch.Tensor  # int32 [experts], zero before every use

    @property
    def num(self) -> int:
        return self.gate_up.shape[0]


def make_experts(router, gates, ups, downs, top: int, limit: float, slope: float, dtype, device) -> Experts:
    """Interleave and stack per-expert gate / up [ff, width] and down [width, ff] matrices."""
    E, (F, W) = len(gates), gates[0].shape
    gate_up = torch.empty(E, F, 2, W, dtype=dtype, device=device)
    down = torch.empty(E, W, F, dtype=dtype, device=device)
    for e in range(E):
        gate_up[e, :, 0] = gates[e].to(device, dtype)
        gate_up[e, :, 1] = ups[e].to(device, dtype)
        down[e] = downs[e].to(device, dtype)
    return Experts(router.to(device, torch.bfloat16).contiguous(), gate_up.view(E, 2 * F, W), down, top, limit, slope,
                   torch.zeros(E, dtype=torch.int32, device=device))


def expert_tile_rows(num_rows: int, top: int, experts: int, dtype) -> int:
    """Most rows of an expert's tile: 256 for prompt-sized steps (the widest tcgen05 tile), 64 for small ones, where
    weights are streamed and a narrow tile leaves shared memory for a deeper ring."""
    if dtype == torch.float32:
        return 32
    # The line lies where some expert begins to have more than 64 rows, whose weights are then read twice; of many experts one does sooner.
    # us a layer with tiles of 64 and 256, rows an expert in brackets: 8 experts of 3072 [53.2] 83.2 and 86.1, [54] 103.0 and 86.2; 12 of 2048
    # [41.7] 85.9 and 84.2, [46.7] 92.7 and 84.9; 16 of 2048 [37.5] 104.3 and 104.5, [42.5] 106.6 and 103.9, [47.5] 116.9 and 104.9; 20 of 1536 [36]
    # 101.1 and 100.5; 24 [33.3] 114.2 and 112.8, [39] 120.9 and 114.3; 32 [36] 138.6 and 137.2, [37.5] 147.1 and 137.4; 64 of 1024 [31.2] 184.2 and 179.7.
    return 64 if num_rows * top <= min(54 * experts, 28 * experts + 200) else 256


def max_expert_tiles(total: int, experts: int, tile_rows: int) -> int:
    return total // tile_rows + min(experts, total)


def one_launch(total: int, experts: int, width: int, ff: int, sms: int) -> bool:
    """Whether both products of the experts are one launch."""
    # Unless the second one's items are the longer ones: as the last to be drawn they leave multiprocessors idle
    # for longer than a start takes.  us a layer, two launches and one: 32 experts of 1536 (width 2048), 64 rows 135.3 and 123.0, 512 154.6
    # and 145.4, 1024 175.2 and 165.7; 8 experts of 3072, 64 rows 79.5 and 82.3, 192 84.4 and 94.1, 700 106.8 and 113.8 (16 80.1 and 77.3, 1000 135 and 129).
    # Not where the first product of all experts is less than two rounds of items (8 experts of 2048, 32 rows 62.3 and 66.4), nor where that of the
    # experts that a few rows can reach is less than one, since the second one's would only wait (1 row, 4 of 32 experts 45.2 and 46.9, 2 rows 63.6
    # and 63.4, 3 rows 72.0 and 66.0; 2 rows, 4 of 64 experts of 1024 45.8 and 46.9, 3 rows 71.6 and 66.5), nor where tiles are full and the
    # tensor core is the bound (32 experts of 1536, router and dispatch included: 1536 rows 175.3 and 173.4, 2048 213.9 and 228.2, 4096 367 and 408).
    items = (2 * ff + 127) // 128  # of an expert with one tile
    return ff <= width and total <= 192 * experts and items * experts >= 2 * sms and items * min(experts, total) >= sms


def grouped_linear(x, w, tiles, max_tiles, tile_rows, scores=None, limit=0.0, slope=0.0, variant: int | None = None):
    """Rows of x (ordered by expert) times their expert's matrix w [E, out, in]; with scores: the gated unit, half as
    many outputs."""
    rows, width = x.shape
    E, out_rows, _ = w.shape
    act = scores is not None
    if variant is None:
        variant = 0 if x.dtype == torch.bfloat16 and width % 8 == 0 else 1
    y = torch.empty(rows, out_rows // 2 if act else out_rows, device=x.device, dtype=x.dtype)
    rc = _lib_dec().b200dec_grouped_linear(
        x.data_ptr(), w.data_ptr(), x.element_size(), tiles.data_ptr(), max_tiles, tile_rows, rows, E, out_rows, width, _ptr(scores),
        int(act), float(limit), float(slope), y.data_ptr(), K.num_sms(x.device), variant, K.status_word(x.device).data_ptr(), K._stream())
    _lib.check(rc, "grouped_linear")
    return y


@K._ranged
def mixture(x: torch.Tensor, xb: torch.Tensor, ex: Experts, variant: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Routed experts of every row.  x: the rows in fp32 (the router's input), xb: in the model's precision.  The score
    multiplies the expert's input.  Returns (outputs [N * top, width] ordered by expert, places int32 [N, top]): the
    layer's output for row r is the sum of outputs[places[r]] (scaled_add_norm takes both).  `ex.counts` must be
    zero, which scaled_add_norm(zero=ex.counts) sees to."""
    K._require_cuda(x, xb, ex.gate_up)
    lib, dev = _lib_dec(), x.device
    N, W = x.shape
    total, E = N * ex.top, ex.num
    tile_rows = expert_tile_rows(N, ex.top, E, xb.dtype)
    max_tiles = max_expert_tiles(total, E, tile_rows)
    # separate allocations: no kernel of the chain reads a cache line that the next one's input shares
    ids, ranks, slots, scores = (torch.empty(total, dtype=torch.int32, device=dev) for _ in range(4))
    tiles = torch.empty(1 + 3 * max_tiles + max_tiles + 1, dtype=torch.int32, device=dev)  # and the counters of the products behind them
    ff = ex.down.shape[2]
    both = variant is None and xb.dtype == torch.bfloat16 and W % 8 == 0 and ff % 8 == 0 and one_launch(total, E, W, ff, K.num_sms(dev))
    done = tiles.data_ptr() + 4 * (1 + 3 * max_tiles) if both else None
    score_sorted = torch.empty(total, dtype=torch.float32, device=dev)
    rc = lib.b200dec_router(x.data_ptr(), ex.router.data_ptr(), N, W, E, ex.top, ids.data_ptr(), scores.data_ptr(), ranks.data_ptr(),
                            ex.counts.data_ptr(), K._stream())
    _lib.check(rc, "router")
    xs = torch.empty(total, W, device=dev, dtype=xb.dtype)
    rc = lib.b200dec_dispatch_counted(xb.data_ptr(), xb.element_size(), ids.data_ptr(), scores.data_ptr(), ranks.data_ptr(), ex.counts.data_ptr(), N,
                                      W, E, ex.top, tile_rows, xs.data_ptr(), score_sorted.data_ptr(), slots.data_ptr(), tiles.data_ptr(), max_tiles,
                                      done, K._stream())
    _lib.check(rc, "dispatch")
    if both:
        h, y = (torch.empty(total, n, device=dev, dtype=xb.dtype) for n in (ff, W))
        rc = lib.b200dec_expert_products(xs.data_ptr(), ex.gate_up.data_ptr(), ex.down.data_ptr(), tiles.data_ptr(), max_tiles, tile_rows, total, E,
                                         ff, W, score_sorted.data_ptr(), float(ex.limit), float(ex.slope), h.data_ptr(), y.data_ptr(),
                                         done, K.num_sms(dev), K.status_word(dev).data_ptr(), K._stream())
        _lib.check(rc, "expert_products")
        return y, slots.view(N, ex.top)
    h = grouped_linear(xs, ex.gate_up, tiles, max_tiles, tile_rows, score_sorted, ex.limit, ex.slope, variant)
    return grouped_linear(h, ex.down, tiles, max_tiles, tile_rows, variant=variant), slots.view(N, ex.top)


# ----------------------------------------------------------------------------- recurrent layers
@dataclass
class Recurrence:
    """Constants of a layer that carries a state S [dim, vdim] per head (include/b200dec.h, b200dec_recurrence):
    S <- decay S; u = beta (v - S^T k) with `correct`, else step * v; S <- S + k u^T; o = S^T q + skip v."""

    heads: int
    qk_heads: int
    dim: int
    vdim: int
    conv_w: torch.Tensor  # fp32 [taps, channels], last row: the current token
    conv_b: torch.Tensor | None  # fp32 [channels]
    neg_a: torch.Tensor  # fp32 [heads]: decay = exp(neg_a * softplus(step_in + dt_bias))
    dt_bias: torch.Tensor  # fp32 [heads], or [heads * dim] with channel_decay
    skip: torch.Tensor | None  # fp32 [heads]
    off_q: int
    off_k: int
    off_v: int
    channel_decay: bool = False
    correct: bool = False
    unit_eps: float | None = None  # unit q and k per head, x / sqrt(sum(x^2) + unit_eps)
    q_scale: float = 1.0

    @property
    def taps(self) -> int:
        return self.conv_w.shape[0]

    @property
    def channels(self) -> int:
        return self.conv_w.shape[1]


@dataclass
class RecurrentState:
    """What a recurrent layer keeps per request slot: the 32-bit state and the convolution's last raw inputs by position."""

    state: torch.Tensor  # fp32 [slots, heads, dim, round4(vdim)]
    ring: torch.Tensor  # [slots, taps, channels]


def make_recurrent_state(rec: Recurrence, slots: int, dtype, device) -> RecurrentState:
    return RecurrentState(torch.zeros(slots, rec.heads, rec.dim, (rec.vdim + 3) // 4 * 4, device=device),
                          torch.zeros(slots, rec.taps, rec.channels, dtype=dtype, device=device))


@dataclass
class GatedNorm:
    """Norm of a row's `parts` equal parts by themselves: times silu(gate) before (gate_first) or sigmoid(gate) after."""

    weight: torch.Tensor  # fp32, repeated along the row
    parts: int
    eps: float
    gate_first: bool
    out_scale: float = 1.0


def _recurrence_args(rec: Recurrence, st: RecurrentState, x, step, beta):
    assert x.stride(1) == 1 and x.shape[1] == rec.channels and x.dtype == st.ring.dtype and step.stride(1) == 1 and step.dtype == x.dtype
    assert st.state.is_contiguous() and st.ring.is_contiguous() and (beta is None or (beta.stride(1) == 1 and beta.dtype == x.dtype))
    assert step.shape[1] == rec.heads * (rec.dim if rec.channel_decay else 1) == rec.dt_bias.numel()
    r = _lib.Recurrence(st.state.data_ptr(), st.ring.data_ptr(), rec.conv_w.data_ptr(), _ptr(rec.conv_b), rec.neg_a.data_ptr(),
                        rec.dt_bias.data_ptr(), _ptr(rec.skip), st.state.shape[0], rec.heads, rec.qk_heads, rec.dim, rec.vdim, rec.taps,
                        x.element_size(), rec.channels, rec.off_q, rec.off_k, rec.off_v, int(rec.channel_decay), int(rec.correct),
                        int(rec.unit_eps is not None), rec.unit_eps or 0.0, rec.q_scale)
    i = _lib.RecurrenceIn(x.data_ptr(), step.data_ptr(), _ptr(beta), x.stride(0), step.stride(0), 0 if beta is None else beta.stride(0))
    return r, i


@K._ranged
def recurrence_decode(rec: Recurrence, st: RecurrentState, x, step, beta, rows: Rows, out: torch.Tensor, norm: GatedNorm | None = None,
                      gate: torch.Tensor | None = None, variant: int = 0) -> None:
    """One token of every decoding entry: convolution, state and read-out; out fp32 [N, heads * vdim], or with `norm` (one part
    per head, gate behind it) the gated output in the model's precision."""
    K._require_cuda(x, out, st.state)
    r, i = _recurrence_args(rec, st, x, step, beta)
    e = rows.entries()
    rc = _lib_dec().b200dec_recurrence_decode(
        ctypes.byref(r), ctypes.byref(i), ctypes.byref(e), None if norm is None else norm.weight.data_ptr(), 0.0 if norm is None else norm.eps,
        _ptr(gate), 0 if gate is None else gate.stride(0), out.data_ptr(), out.stride(0), variant, K.num_sms(x.device),
        K.status_word(x.device).data_ptr(), K._stream())
    _lib.check(rc, "recurrence_decode")


@K._ranged
def conv_rows(rec: Recurrence, st: RecurrentState, x, step, beta, rows: Rows) -> torch.Tensor:
    """silu(convolution) of the prompt portions' rows, all channels."""
    K._require_cuda(x, st.ring)
    r, i = _recurrence_args(rec, st, x, step, beta)
    e = rows.entries()
    conv = torch.empty(rows.num_rows, _round8(rec.channels), device=x.device, dtype=x.dtype)
    rc = _lib_dec().b200dec_conv_rows(ctypes.byref(r), ctypes.byref(i), ctypes.byref(e), conv.data_ptr(), K.status_word(x.device).data_ptr(),
                                      K._stream())
    _lib.check(rc, "conv_rows")
    return conv


@K._ranged
def recurrence_prefill(rec: Recurrence, st: RecurrentState, x, step, beta, rows: Rows, out: torch.Tensor, form: str | None = None) -> None:
    """The prompt portions' rows: convolution, then the state through every portion; out fp32 [N, heads * vdim].  `form`: which
    kernel carries the state ("scan" token by token, any sizes; "blocked", "chunked"); default: the fastest that applies."""
    K._require_cuda(x, out, st.state)
    conv = conv_rows(rec, st, x, step, beta, rows)
    r, i = _recurrence_args(rec, st, x, step, beta)
    e = rows.entries()
    lib, status = _lib_dec(), K.status_word(x.device).data_ptr()
    sizes = {"chunked": lib.b200dec_state_space_chunked_workspace(ctypes.byref(r)),
             "blocked": lib.b200dec_recurrence_blocked_workspace(ctypes.byref(r), ctypes.byref(e)) if rec.skip is None else 0}
    if form is None:
        form = next((f for f, n in sizes.items() if n), "scan")
    if form == "scan":
        rc = lib.b200dec_recurrence_scan(ctypes.byref(r), ctypes.byref(i), conv.data_ptr(), ctypes.byref(e), out.data_ptr(), status, K._stream())
    else:
        ws = torch.empty(sizes[form], dtype=torch.uint8, device=x.device)
        args = (ctypes.byref(r), ctypes.byref(i), conv.data_ptr(), ctypes.byref(e), out.data_ptr(), ws.data_ptr(), sizes[form])
        if form == "chunked":
            rc = lib.b200dec_state_space_chunked(*args, K.num_sms(x.device), status, K._stream())
        else:
            rc = lib.b200dec_recurrence_blocked(*args, status, K._stream())
    _lib.check(rc, f"recurrence_{form}")


@K._ranged
def gated_norm(o: torch.Tensor, gate: torch.Tensor, norm: GatedNorm, out: torch.Tensor) -> None:
    K._require_cuda(o, gate, out)
    assert o.is_contiguous() and o.dtype == torch.float32 and gate.stride(1) == 1 and gate.dtype == out.dtype and out.stride(1) == 1
    assert gate.shape == o.shape == out.shape and norm.weight.dtype == torch.float32
    rc = _lib_dec().b200dec_gated_norm(o.data_ptr(), gate.data_ptr(), gate.stride(0), int(norm.gate_first), out.element_size(),
                                       norm.weight.data_ptr(), norm.weight.numel(), norm.eps, norm.out_scale, out.data_ptr(), out.stride(0),
                                       o.shape[0], o.shape[1], norm.parts, K._stream())
    _lib.check(rc, "gated_norm")


def recurrent_mixer(rec: Recurrence, st: RecurrentState, x, step, beta, gate, norm: GatedNorm, rows: Rows, out: torch.Tensor) -> None:
    """A recurrent layer between its projections: out [N, heads * vdim] in the model's precision."""
    if rows.seq_ids is None and not norm.gate_first and norm.parts == rec.heads and norm.weight.numel() == rec.vdim and norm.out_scale == 1.0:
        return recurrence_decode(rec, st, x, step, beta, rows, out, norm, gate)
    o = torch.empty(x.shape[0], rec.heads * rec.vdim, device=x.device, dtype=torch.float32)
    recurrence_decode(rec, st, x, step, beta, rows, o)
    if rows.seq_ids is not None:
        recurrence_prefill(rec, st, x, step, beta, rows, o)
    gated_norm(o, gate, norm, out)


# ----------------------------------------------------------------------------- projections side by side
class Packed:
    """Matrices with a common input as one product.  Every part starts at a multiple of 8 output channels, so that the parts
    of a row can be read in vectors."""

    def __init__(self, parts: dict[str, torch.Tensor], dtype, device):
        self.at: dict[str, tuple[int, int]] = {}
        blocks, n = [], 0
        for name, w in parts.items():
            self.at[name] = (n, n + w.shape[0])
            pad = -w.shape[0] % 8
            blocks.append(w.to(device, dtype))
            if pad:
                blocks.append(torch.zeros(pad, w.shape[1], dtype=dtype, device=device))
            n += w.shape[0] + pad
        self.weight = torch.cat(blocks)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return K.linear(x, self.weight)

    def part(self, y: torch.Tensor, name: str) -> torch.Tensor:
        lo, hi = self.at[name]
        return y[:, lo:hi]


# ----------------------------------------------------------------------------- low-rank adapters of many requests
MAX_ADAPTER_RANK = 128


@dataclass(frozen=True, eq=False)
class Adapters:
    """Low-rank adapters of one shared projection, a slot each: y + scale[a] * (x down[a]^T) up[a]^T.  `parts`: the projection's columns, one number
    for each part that has a product of its own (query, key, value of a packed one); rows p * rank .. of down belong to part p."""

    down: torch.Tensor  # [slots, parts * rank, width]
    up: torch.Tensor  # [slots, out, rank]
    scale: torch.Tensor  # fp32 [slots]
    parts: tuple[int, ...]

    def __post_init__(self):
        d, u, s, parts = self.down, self.up, self.scale, tuple(self.parts)
        if d.dim() != 3 or u.dim() != 3 or s.dim() != 1 or not d.is_contiguous() or not u.is_contiguous() or not s.is_contiguous():
            raise ValueError("adapters: contiguous down [slots, parts * rank, width], up [slots, out, rank] and scale [slots] are wanted")
        slots, out, rank = u.shape
        if not 1 <= len(parts) <= 4 or min(parts) < 1 or sum(parts) != out:
            raise ValueError(f"adapters: one to four parts that add up to the {out} columns, not {parts}")
        if rank % 8 or not 8 <= rank <= MAX_ADAPTER_RANK:
            raise ValueError(f"adapters: the rank is a multiple of 8 up to {MAX_ADAPTER_RANK}, not {rank}")
        if not 1 <= slots <= 4096 or d.shape[:2] != (slots, len(parts) * rank) or s.shape[0] != slots or d.shape[2] < 1:
            raise ValueError(f"adapters: down {tuple(d.shape)} and scale {tuple(s.shape)} do not fit up {tuple(u.shape)} of {len(parts)} parts")
        if d.dtype != u.dtype or s.dtype != torch.float32 or not d.device == u.device == s.device:
            raise ValueError("adapters: down and up of one type, a 32-bit scale, all on one device")
        ends = [sum(parts[: i + 1]) for i in range(len(parts))]
        st = _lib.Adapters(d.data_ptr(), u.data_ptr(), s.data_ptr(), slots, rank, d.shape[2], len(parts), _elem(d.dtype))
        st.ends[: len(ends)] = ends
        for name, value in dict(parts=parts, struct=st, ref=ctypes.byref(st), slots=slots, out=out, rank=rank, width=d.shape[2], dtype=u.dtype,
                                device_index=u.get_device()).items():
            object.__setattr__(self, name, value)

    def load(self, slot: int, pairs, scale: float) -> None:
        """Put an adapter into a slot: a pair (down [r, width], up [columns of the part, r]) for each part, r up to the rank, or None for a part that
        it leaves alone."""
        if not 0 <= slot < self.slots or len(pairs) != len(self.parts):
            raise ValueError(f"adapters: slot {slot} of {self.slots}, {len(pairs)} pairs for {len(self.parts)} parts")
        for pair, n in zip(pairs, self.parts):
            if pair is not None and (pair[0].dim() != 2 or pair[0].shape[0] > self.rank or pair[0].shape[1] != self.width
                                     or tuple(pair[1].shape) != (n, pair[0].shape[0])):
                raise ValueError(f"adapters: {tuple(pair[0].shape)} and {tuple(pair[1].shape)} for {self.width} inputs, {n} columns and "
                                 f"ranks up to {self.rank}")
        self.clear(slot)
        at = 0
        for i, (pair, n) in enumerate(zip(pairs, self.parts)):
            if pair is not None:
                r = pair[0].shape[0]
                self.down[slot, i * self.rank : i * self.rank + r] = pair[0].to(self.down)
                self.up[slot, at : at + n, :r] = pair[1].to(self.up)
            at += n
        self.scale[slot] = float(scale)

    def clear(self, slot: int) -> None:
        """An adapter that adds nothing."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"adapters: slot {slot} of {self.slots}")
        self.down[slot] = 0
        self.up[slot] = 0
        self.scale[slot] = 0


def make_adapters(slots: int, width: int, parts, rank: int, dtype, device) -> Adapters:
    """Empty slots for adapters of up to `rank` (rounded up to a multiple of 8) beside a projection of `width` inputs."""
    rank = _round8(rank)
    return Adapters(torch.zeros(slots, len(parts) * rank, width, dtype=dtype, device=device),
                    torch.zeros(slots, sum(parts), rank, dtype=dtype, device=device), torch.zeros(slots, device=device), tuple(parts))


class AdapterPlan:
    """A step's rows sorted by adapter (plan_adapters), for all the projections of the step."""

    def __init__(self, buf: torch.Tensor, rows: int, slots: int, tiles: int, tile_rows: int):
        self.buf, self.rows, self.slots, self.num_tiles, self.tile_rows = buf, rows, slots, tiles, tile_rows
        self.device_index = buf.get_device()
        self.status = K.status_word(buf.device).data_ptr()
        at = buf.data_ptr()
        self.struct = _lib.AdapterPlan(at + 16 * tiles, at, tiles, tile_rows, rows, slots)
        self.ref = ctypes.byref(self.struct)

    @property
    def tiles(self) -> torch.Tensor:
        """int32 [tiles, 4]: adapter (-1: none) and number of rows; the first one's third number: tiles that have rows."""
        return self.buf[: 4 * self.num_tiles].view(self.num_tiles, 4)

    @property
    def order(self) -> torch.Tensor:
        """int32 [tiles, tile_rows]: the rows of each tile, -1 behind them."""
        return self.buf[4 * self.num_tiles :].view(self.num_tiles, self.tile_rows)


def adapter_tile_rows(num_rows: int) -> int:
    """Rows of a tile: 16 for decoding rows, 128 where rows of one adapter come in portions.

    Measured, the four projections [2048 -> 4096], [2048 -> 2048], [2048 -> 12288] and [6144 -> 2048] together, tiles of 16 and of 128: 256 rows of 48 adapters
    of rank 16 44 and 57 us, of 4 adapters of rank 16 28 and 31 us, of rank 64 73 and 60 us; 512 rows of 4 adapters of rank 32 65 and 56 us, of rank 64 115 and
    61 us."""
    return 16 if num_rows <= 256 else 128


def _here(t: torch.Tensor) -> None:
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on {t.device} while device {torch.cuda.current_device()} is the current one")


@K._ranged
def plan_adapters(ids: torch.Tensor, slots: int, tile_rows: int | None = None) -> AdapterPlan:
    """Sort a step's rows by adapter.  ids int32 [rows]: each row's slot, -1: none; others outside [0, slots) count as that and set a status bit.  One launch per
    step, for every add_adapters of it."""
    dev = ids.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        K._require_cuda(ids)
        _here(ids)
    if ids.dtype != torch.int32 or ids.dim() != 1 or not ids.is_contiguous():
        raise ValueError("plan_adapters: contiguous int32 ids [rows] are wanted")
    if not 1 <= slots <= 4096:
        raise ValueError(f"plan_adapters: 1 to 4096 slots, not {slots}")
    N = ids.shape[0]
    rows = adapter_tile_rows(N) if tile_rows is None else tile_rows
    if rows not in (16, 128):
        raise ValueError(f"plan_adapters: tiles of 16 or 128 rows, not {rows}")
    most = N // rows + min(N, slots + 1)
    plan = AdapterPlan(ids.new_empty((4 + rows) * most), N, slots, most, rows)
    rc = _lib_dec().b200dec_adapter_plan(ids.data_ptr(), plan.ref, plan.status, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, "plan_adapters")
    return plan


@K._ranged
def add_adapters(y: torch.Tensor, x: torch.Tensor, adapters: Adapters, plan: AdapterPlan, out: torch.Tensor | None = None) -> torch.Tensor:
    """y + scale * (x down^T) up^T of every row's adapter; rows without one stay y.  y [rows, out]: what the shared projection made of x [rows, width].
    Written over y unless `out` is given, which shares no memory with y or x."""
    if out is None:
        out = y
    N, dtype, dev = plan.rows, adapters.dtype, plan.device_index
    if not y.get_device() == x.get_device() == out.get_device() == adapters.device_index == dev:
        K._require_cuda(y, x, out, adapters.up)
        raise ValueError("add_adapters: rows, adapters and plan on one device are wanted")
    if dev != torch._C._cuda_getDevice():
        _here(y)
    if not y.dtype is x.dtype is out.dtype is dtype:
        raise ValueError(f"add_adapters: rows of {x.dtype}, {y.dtype} and {out.dtype} beside adapters of {dtype}")
    wide = (N, adapters.out)
    if x.shape != (N, adapters.width) or y.shape != wide or out.shape != wide:
        raise ValueError(f"add_adapters: {tuple(x.shape)}, {tuple(y.shape)} and {tuple(out.shape)} for a plan of {N} rows")
    if plan.slots != adapters.slots:
        raise ValueError(f"add_adapters: a plan for {plan.slots} slots and {adapters.slots} adapters")
    if N > 1:
        (xs, x1), (ys, y1), (os, o1) = x.stride(), y.stride(), out.stride()
        if not x1 == y1 == o1 == 1:
            raise ValueError("add_adapters: a row's elements lie side by side")
    else:  # a single row's stride may be anything
        if N and not x.stride(1) == y.stride(1) == out.stride(1) == 1:
            raise ValueError("add_adapters: a row's elements lie side by side")
        xs, ys, os = _round8(adapters.width), _round8(adapters.out), _round8(adapters.out)
    lib, ws, nbytes = _lib_dec(), None, 0
    if plan.tile_rows > 16:
        nbytes = lib.b200dec_add_adapters_workspace(adapters.ref, plan.ref)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=y.device)
    rc = lib.b200dec_add_adapters(adapters.ref, plan.ref, x.data_ptr(), xs, y.data_ptr(), ys, out.data_ptr(), os, None if ws is None else ws.data_ptr(), nbytes,
                                  plan.status, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, "add_adapters")
    return out


# ----------------------------------------------------------------------------- what requests ask of their next token
MAX_CHOICE_VOCAB = 393216


def _entries_of(what: str, tensors: dict) -> int | None:
    """The common length of a record's per-entry tensors (contiguous, on one device); None if it has none."""
    n = None
    for name, (t, dtype) in tensors.items():
        if t is None:
            continue
        if t.dtype != dtype or t.dim() < 1 or not t.is_contiguous():
            raise ValueError(f"{what}: {name} is a contiguous tensor of {dtype} with an element or a row per entry, not {t.dtype} {tuple(t.shape)}")
        if n is not None and t.shape[0] != n:
            raise ValueError(f"{what}: {name} has {t.shape[0]} entries, others {n}")
        n = t.shape[0]
    return n


@dataclass(frozen=True, eq=False)
class Rules:
    """Penalties for repeated tokens, biases and grammar masks of a step's entries (include/b200dec.h, b200dec_rules).  Per entry: slots, its row of the
    history (-1: passed over), lengths, tokens there, and prompts, how many of them are the prompt (int32); repetition (1: none), presence,
    frequency (fp32); bias_ids int32 and bias fp32 [entries, n] (id -1: unused); mask_rows int32, its row of masks, -1: none."""

    history: torch.Tensor | None = None  # int32 [requests, capacity]
    slots: torch.Tensor | None = None
    lengths: torch.Tensor | None = None
    prompts: torch.Tensor | None = None
    repetition: torch.Tensor | None = None
    presence: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    masks: torch.Tensor | None = None  # int32 [masks, words of 32 tokens]
    mask_rows: torch.Tensor | None = None

    def __post_init__(self):
        i, f = torch.int32, torch.float32
        per_entry = {"slots": (self.slots, i), "lengths": (self.lengths, i), "prompts": (self.prompts, i), "repetition": (self.repetition, f),
                     "presence": (self.presence, f), "frequency": (self.frequency, f), "bias_ids": (self.bias_ids, i), "bias": (self.bias, f),
                     "mask_rows": (self.mask_rows, i)}
        n = _entries_of("rules", per_entry)
        for name, (t, _) in per_entry.items():
            if t is not None and t.dim() != (2 if name.startswith("bias") else 1):
                raise ValueError(f"rules: {name} {tuple(t.shape)} has the wrong number of dimensions")
        for name in ("history", "masks"):
            t = getattr(self, name)
            if t is not None and (t.dtype != i or t.dim() != 2 or not t.is_contiguous()):
                raise ValueError(f"rules: {name} is a contiguous int32 matrix")
        if (self.history is None) != (self.lengths is None) or (self.history is None and self.prompts is not None):
            raise ValueError("rules: a history, lengths and prompts belong together")
        if self.history is None and any(t is not None for t in (self.repetition, self.presence, self.frequency)):
            raise ValueError("rules: penalties need a history")
        if (self.bias is None) != (self.bias_ids is None) or (self.bias is not None and self.bias.shape != self.bias_ids.shape):
            raise ValueError("rules: as many biases as tokens for them")
        if (self.masks is None) != (self.mask_rows is None):
            raise ValueError("rules: masks and the entries' rows of them belong together")
        tensors = [t for t in vars(self).values() if t is not None]
        if len({t.device for t in tensors}) > 1:
            raise ValueError("rules: tensors on several devices")
        h, m = self.history, self.masks
        object.__setattr__(self, "entries", n)
        object.__setattr__(self, "device_index", tensors[0].get_device() if tensors else None)
        object.__setattr__(self, "struct", _lib.Rules(
            _ptr(h), _ptr(self.slots), _ptr(self.lengths), _ptr(self.prompts), _ptr(self.repetition), _ptr(self.presence), _ptr(self.frequency),
            _ptr(self.bias_ids), _ptr(self.bias), _ptr(m), _ptr(self.mask_rows), 0 if h is None else h.shape[1], 0 if h is None else h.shape[0],
            0 if self.bias is None else self.bias.shape[1], 0 if m is None else m.shape[0], 0 if m is None else m.shape[1]))
        object.__setattr__(self, "ref", ctypes.byref(self.struct))


@dataclass(frozen=True, eq=False)
class Draw:
    """How a step's entries draw their tokens (include/b200dec.h, b200dec_draw), a number per entry: temperature (0: the largest logit), uniform
    in [0, 1), top_k (int32, 0: all), top_p (1: all), min_p (0: all; a token's weight beside the most likely one's)."""

    temperature: torch.Tensor
    uniform: torch.Tensor
    top_k: torch.Tensor | None = None
    top_p: torch.Tensor | None = None
    min_p: torch.Tensor | None = None

    def __post_init__(self):
        i, f = torch.int32, torch.float32
        n = _entries_of("draw", {"temperature": (self.temperature, f), "uniform": (self.uniform, f), "top_k": (self.top_k, i),
                                 "top_p": (self.top_p, f), "min_p": (self.min_p, f)})
        tensors = [t for t in vars(self).values() if t is not None]
        if any(t.dim() != 1 for t in tensors) or len({t.device for t in tensors}) > 1:
            raise ValueError("draw: one number per entry, all on one device")
        object.__setattr__(self, "entries", n)
        object.__setattr__(self, "device_index", self.uniform.get_device())
        object.__setattr__(self, "struct", _lib.Draw(*(_ptr(t) for t in (self.temperature, self.top_k, self.top_p, self.min_p, self.uniform))))
        object.__setattr__(self, "ref", ctypes.byref(self.struct))


def _check_logits(what: str, logits: torch.Tensor, rules: Rules | None) -> tuple[int, int, int, int]:
    """Entries, vocabulary, row stride and element size of a step's logits."""
    dev = logits.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        K._require_cuda(logits)
        _here(logits)
    elem = 2 if logits.dtype == torch.bfloat16 else 4 if logits.dtype == torch.float32 else 0
    if logits.dim() != 2 or not elem or not logits.shape[1]:
        raise ValueError(f"{what}: bf16 or fp32 logits [entries, vocab] are wanted")
    (E, V), (stride, one) = logits.shape, logits.stride()
    if V > 1 and one != 1:
        raise ValueError(f"{what}: a row's logits lie side by side")
    if rules is not None:
        if rules.entries is not None and rules.entries != E:
            raise ValueError(f"{what}: rules for {rules.entries} entries and logits of {E}")
        if rules.device_index is not None and rules.device_index != dev:
            raise ValueError(f"{what}: rules on another device than the logits")
        st = rules.struct
        if st.history and not st.slots and st.num_histories < E:
            raise ValueError(f"{what}: {st.num_histories} histories for {E} entries")
        if st.masks and st.mask_words < (V + 31) // 32:
            raise ValueError(f"{what}: masks of {st.mask_words} words for {V} tokens")
    return E, V, stride if E > 1 else _round8(V), elem  # (a single row's stride may be anything)


@K._ranged
def adjust_logits(logits: torch.Tensor, rules: Rules, out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits [entries, vocab] under each entry's rules, fp32.  `out`: where they go, fp32 logits themselves perhaps; rows of entries that are passed
    over are left there as they are (uninitialised without it)."""
    E, V, stride, elem = _check_logits("adjust_logits", logits, rules)
    if out is None:
        out = logits.new_empty(E, V, dtype=torch.float32)
    elif out.dtype != torch.float32 or out.shape != logits.shape or (V > 1 and out.stride(1) != 1) or out.device != logits.device:
        raise ValueError("adjust_logits: fp32 rows of the logits' shape are wanted")
    rc = _lib_dec().b200dec_adjust_logits(logits.data_ptr(), stride, elem, rules.ref, out.data_ptr(),
                                          out.stride(0) if E > 1 else _round8(V), E, V, K.status_word(logits.device).data_ptr(), K._stream())
    if rc:
        _lib.check(rc, "adjust_logits")
    return out


@K._ranged
def choose_tokens(logits: torch.Tensor, draw: Draw, rules: Rules | None = None, append: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Every entry's next token under its rules and its way of drawing: (int64 [entries], its log-probability under the softmax of the adjusted
    logits, fp32 [entries]); (-1, -inf) where nothing is allowed or the entry is passed over.  append: the token goes behind the entry's
    history where there is room; the entries' rows are different ones then."""
    E, V, stride, elem = _check_logits("choose_tokens", logits, rules)
    if draw.entries != E or draw.device_index != logits.get_device():
        raise ValueError(f"choose_tokens: a draw for {draw.entries} entries on {draw.uniform.device}, logits of {E} on {logits.device}")
    if V > MAX_CHOICE_VOCAB:
        raise ValueError(f"choose_tokens: {V} tokens, at most {MAX_CHOICE_VOCAB}")
    if append and (rules is None or rules.history is None):
        raise ValueError("choose_tokens: nowhere to append to")
    tokens, logprobs = draw.uniform.new_empty(E, dtype=torch.int64), draw.uniform.new_empty(E)
    rc = _lib_dec().b200dec_choose_tokens(logits.data_ptr(), stride, elem, None if rules is None else rules.ref, draw.ref, E, V, int(append),
                                          tokens.data_ptr(), logprobs.data_ptr(), K.status_word(logits.device).data_ptr(), K._stream())
    if rc:
        _lib.check(rc, "choose_tokens")
    return tokens, logprobs
