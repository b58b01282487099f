"""Python face of the kernels of quantised serving (library "quant"): rows and weights in 8 bits with a scale each, their
product, and keys and values held in 4 bits with the attention that reads them.

A row in 8 bits: scale = float32(max |x| / 127), codes x / scale to the nearest integer, ties to even. A row of zeros has a
scale of 0; one with an infinity or a NaN has a scale of NaN, and so are its products. A group of 32 numbers of a head in 4
bits: m the number of largest magnitude (the positive one of two), d = bfloat16(m / -8), codes x / d to the nearest integer, ties to
even, clamped to -8..7; the number stands for code * d. (The layout is in csrc/quant.cuh.)
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from . import ops, sm100

_P = c_void_p
ops.register_signatures("quant", {
    "rllm_quantize_rows": [c_int, _P, c_longlong, _P, _P, c_int, c_float, _P, c_longlong, _P, c_int, c_int, c_int, _P],
    "rllm_int8_gemm": [c_int, c_int, _P, _P, _P, _P, _P, c_longlong, c_int, c_int, c_int, _P, c_int, _P],
    "rllm_kv4_store": [c_int, _P, _P, c_longlong, c_longlong, _P, _P, _P, _P, _P, c_longlong, c_int, c_int, c_int, c_int, _P],
    "rllm_kv4_read": [c_int, _P, _P, _P, _P, c_longlong, _P, c_int, _P, _P, c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, c_int, c_int,
                      c_int, _P],
    "rllm_kv4_decode": [_P, c_int, _P, _P, _P, _P, c_longlong, _P, c_int, _P, _P, c_int, c_int, c_int, c_int, c_int, c_int, c_float, c_int,
                        c_int, _P],
    "rllm_kv4_attention_simt": [c_int, _P, c_int, _P, _P, _P, _P, c_longlong, _P, c_int, _P, _P, _P, c_int, c_int, c_int, c_int, c_int,
                                c_int, c_float, c_int, _P],
})

INT8_MAX_K = 131072           # 127^2 K stays below 2^31
HEAD_SIZES = (64, 128, 192, 256)


def _here(t: torch.Tensor, name: str) -> None:
    """The launch goes to the current device's current stream: a tensor of another device would be read from there."""
    ops._cuda(t, name)
    if t.device.index != ops._raw_device():
        raise ops.KernelError(f"{name} is on {t.device}, the current device is cuda:{ops._raw_device()}")


class Int8Rows:
    """Rows in 8 bits: `codes` int8 [rows, width rounded up to a multiple of 16] (zeros behind the width), `scales` float32
    [rows]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, width: int):
        self.codes, self.scales, self.width = codes, scales, int(width)

    @property
    def shape(self):
        return (self.codes.shape[0], self.width)

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def dequantize(self) -> torch.Tensor:
        """The numbers the codes stand for, float32."""
        return self.codes[:, : self.width].float() * self.scales[:, None]


class Int8Matrix(Int8Rows):
    """A weight [N, K] in 8 bits, a scale per output channel: the backend's products take it where they take a tensor."""


def quantize_rows(x: torch.Tensor, norm: tuple | None = None, rows: torch.Tensor | None = None, cls=Int8Rows) -> Int8Rows:
    """Rows of x [T, K] (float32 or bfloat16, unit inner stride) in 8 bits. `norm` (weight, eps): of their RMSNorm, which is not
    rounded in between. `rows` int32 [R]: of those rows only."""
    _here(x, "x")
    dt = ops._dt(x, "x")
    if x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ops.KernelError("quantize_rows takes [T, K] rows with unit inner stride")
    T, K = x.shape
    if K < 1:
        raise ops.KernelError("quantize_rows: rows without numbers")
    if rows is not None:
        _here(rows, "rows")
        if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous():
            raise ops.KernelError("quantize_rows: rows must be a contiguous int32 vector")
        T = rows.numel()
    w, eps = norm if norm is not None else (None, 0.0)
    if w is not None:
        _here(w, "norm weight")
        if w.shape != (K,) or not w.is_contiguous():
            raise ops.KernelError(f"norm weight must be a contiguous [{K}], got {tuple(w.shape)}")
    codes = torch.empty((T, (K + 15) // 16 * 16), dtype=torch.int8, device=x.device)
    scales = torch.empty(T, dtype=torch.float32, device=x.device)
    ops._check(ops._fn("quant", "rllm_quantize_rows")(
        dt, x.data_ptr(), x.stride(0), ops._ptr(rows), ops._ptr(w), 0 if w is None else ops._dt(w, "norm weight"), float(eps),
        codes.data_ptr(), codes.stride(0), scales.data_ptr(), T, K, int(cls is Int8Rows), ops._stream()), "quantize_rows")
    return cls(codes, scales, K)


def quantize_matrix(w: torch.Tensor) -> Int8Matrix:
    """A weight [N, K] in 8 bits, a scale per row (output channel)."""
    return quantize_rows(w, cls=Int8Matrix)


def linear_int8(x: Int8Rows, w: Int8Matrix, epilogue: int = ops.EPI_STORE, out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x w^T from the codes: the integer sums are exact, times both scales in float. `epilogue`: `ops.EPI_STORE` (rounded once to
    out_dtype), `EPI_STORE_F32`, `EPI_ACCUM_F32` (added into the float `out`) or `EPI_SWIGLU` (w = [gate; up])."""
    if not isinstance(x, Int8Rows) or not isinstance(w, Int8Matrix):
        raise ops.KernelError("linear_int8 takes Int8Rows and an Int8Matrix")
    _here(x.codes, "x"); _here(w.codes, "w")
    T, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ops.KernelError(f"linear_int8: x has {K} columns, w has {w.shape[1]}")
    if K > INT8_MAX_K:
        raise ops.KernelError(f"linear_int8: {K} columns; the sums are exact in 32 bits up to {INT8_MAX_K}")
    if epilogue not in (ops.EPI_STORE, ops.EPI_STORE_F32, ops.EPI_ACCUM_F32, ops.EPI_SWIGLU):
        raise ops.KernelError(f"linear_int8 has no epilogue {epilogue}")
    if epilogue == ops.EPI_SWIGLU:
        if N % 2:
            raise ops.KernelError("linear_int8: a gate/up pair has an even number of rows")
        N //= 2
    want = torch.float32 if epilogue in (ops.EPI_STORE_F32, ops.EPI_ACCUM_F32) else out_dtype
    if out is None:
        if epilogue == ops.EPI_ACCUM_F32:
            raise ops.KernelError("linear_int8: nothing to add into (`out`)")
        out = torch.empty((T, N), dtype=want, device=x.device)
    _here(out, "out")
    if tuple(out.shape) != (T, N) or out.dtype != want or (out.stride(1) != 1 and N > 1) or (T > 1 and out.stride(0) < N):
        raise ops.KernelError(f"linear_int8: out must be {want} [{T}, {N}] with unit inner stride and rows side by side")
    st = sm100.init(x.device)
    ops._check(ops._fn("quant", "rllm_int8_gemm")(
        epilogue, ops._dt(out, "out"), x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(),
        max(out.stride(0), N), T, N, x.codes.shape[1], st.err.data_ptr(), st.sm_count, ops._stream()), "linear_int8")
    return out


# ---------------------------------------------------------------------------------------------
# keys and values held in 4 bits

def _kv4(tensors: dict) -> tuple:
    """(k4, ks, v4, vs, pages, kv heads, page size, head size) of a layer's tensors, checked."""
    k4, ks, v4, vs = (tensors[n] for n in ("k4", "ks", "v4", "vs"))
    pages, nkv, page_size, half = k4.shape
    hd = 2 * half
    if hd not in HEAD_SIZES:
        raise ops.KernelError(f"a cache held in 4 bits has heads of {HEAD_SIZES}, not {hd}")
    for t, name, dt, n in ((k4, "k4", torch.uint8, half), (v4, "v4", torch.uint8, half), (ks, "ks", torch.bfloat16, hd // 32),
                           (vs, "vs", torch.bfloat16, hd // 32)):
        _here(t, name)
        if t.dtype != dt or tuple(t.shape) != (pages, nkv, page_size, n) or not t.is_contiguous():
            raise ops.KernelError(f"{name} must be contiguous {dt} [{pages}, {nkv}, {page_size}, {n}]")
    return k4, ks, v4, vs, pages, nkv, page_size, hd


def _i32(t: torch.Tensor, name: str, n: int) -> None:
    _here(t, name)
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.numel() < n:
        raise ops.KernelError(f"{name} must be a contiguous int32 vector of at least {n}")


def _table(t: torch.Tensor, rows: int) -> None:
    _here(t, "block_table")
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] < rows or t.stride(1) != 1:
        raise ops.KernelError(f"block_table must be int32 [>= {rows}, pages] with unit inner stride")


def kv4_store(k: torch.Tensor, v: torch.Tensor, tensors: dict, slots: torch.Tensor) -> None:
    """Keys and values [T, kv heads * head size] (float32 or bfloat16, rows may lie apart) into the pages at slots int32 [T]
    (page * page size + offset; -1: not stored). A slot may stand in a call once."""
    k4, ks, v4, vs, pages, nkv, page_size, hd = _kv4(tensors)
    for t, name in ((k, "k"), (v, "v")):
        _here(t, name)
        if t.dim() != 2 or t.shape[1] != nkv * hd or t.stride(1) != 1 or t.shape[0] != k.shape[0] or t.dtype != k.dtype:
            raise ops.KernelError(f"kv4_store: {name} must be [T, {nkv * hd}] with unit inner stride, k and v alike")
    T = k.shape[0]
    _i32(slots, "slots", T)
    ops._check(ops._fn("quant", "rllm_kv4_store")(
        ops._dt(k, "k"), k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), slots.data_ptr(), k4.data_ptr(), ks.data_ptr(),
        v4.data_ptr(), vs.data_ptr(), pages, T, nkv, page_size, hd, ops._stream()), "kv4_store")


def kv4_read(tensors: dict, block_table: torch.Tensor, kv_lens: torch.Tensor, max_kv_len: int,
             dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds for the sequences, as numbers: k, v [S, pages of max_kv_len, kv heads, page size, head size] in dtype
    (float32: exactly code * scale; bfloat16: rounded once). Places behind a sequence's kv_lens, and pages it has given back, are
    zeros."""
    k4, ks, v4, vs, pages, nkv, page_size, hd = _kv4(tensors)
    S = kv_lens.numel()
    _i32(kv_lens, "kv_lens", S)
    _table(block_table, S)
    width = -(-int(max_kv_len) // page_size)
    if width > block_table.shape[1]:
        raise ops.KernelError(f"kv4_read: {max_kv_len} positions are {width} pages, the table has {block_table.shape[1]}")
    k, v = (torch.empty((S, width, nkv, page_size, hd), dtype=dtype, device=k4.device) for _ in range(2))
    ops._check(ops._fn("quant", "rllm_kv4_read")(
        ops._dt(k, "k"), k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, block_table.data_ptr(),
        block_table.stride(0), kv_lens.data_ptr(), None, 0, S, width, page_size, k.data_ptr(), v.data_ptr(), None, None, None, nkv, page_size, hd,
        ops._stream()), "kv4_read")
    return k, v


def _queries(q, nh, nkv, hd, T):
    _here(q, "q")
    if nh <= 0 or nh % nkv or q.dim() != 2 or q.shape[0] != T or q.shape[1] != nh * hd or q.stride(1) != 1:
        raise ops.KernelError(f"attention over 4 bits: q must be [{T}, heads * {hd}] with unit inner stride, heads a multiple of {nkv}")


def attention_kv4_simt(q: torch.Tensor, tensors: dict, token_seq: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
                       nh: int, scale: float, window: int | None = None) -> torch.Tensor:
    """Attention over 4 bits on the CUDA cores, in float: any rows, both run types, every head size."""
    k4, ks, v4, vs, pages, nkv, page_size, hd = _kv4(tensors)
    T = q.shape[0]
    _queries(q, nh, nkv, hd, T)
    _i32(token_seq, "token_seq", T); _i32(positions, "positions", T)
    _table(block_table, 0)
    out = torch.empty((T, nh * hd), dtype=q.dtype, device=q.device)
    ops._check(ops._fn("quant", "rllm_kv4_attention_simt")(
        ops._dt(q, "q"), q.data_ptr(), q.stride(0), k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, out.data_ptr(),
        out.stride(0), token_seq.data_ptr(), positions.data_ptr(), block_table.data_ptr(), block_table.stride(0), T, nh, nkv, hd,
        page_size, float(scale), int(window or 0), ops._stream()), "attention_kv4_simt")
    return out


DECODE_MAX_SPLITS = 8
# Places of a key range's page in the scratch that portions are read into, and bytes of scratch a run of portions may take at once
READ_PAGE, READ_BYTES = 128, 2 << 30


def decode_splits(num_seqs: int, ctas: int, max_kv_len: int, sm_count: int, hd: int) -> int:
    """Ranges the keys of a sequence are cut into (= CTAs of a cluster)."""
    base, best, cost = max(1, num_seqs * ctas), 1, None
    for s in range(1, DECODE_MAX_SPLITS + 1):
        if s > 1 and max_kv_len < 128 * s:
            break
        c = -(-base * s // (2 * sm_count)) * (1150 + max_kv_len * hd / 128 / s) + 50 * s + (200 if s > 1 else 0)
        if cost is None or c < cost:
            best, cost = s, c
    return best


def decode_supported(q: torch.Tensor, hd: int, scale: float) -> bool:
    """Does the tensor-core kernel for single tokens take these queries?"""
    return q.dtype == torch.bfloat16 and hd in (64, 128) and scale > 0 and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0


def attention_kv4_decode(q: torch.Tensor, tensors: dict, kv_lens: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float,
                         window: int | None, max_kv_len: int, splits: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over 4 bits for one bfloat16 query row per sequence, heads of 64 or 128. `max_kv_len`: the most keys of a sequence;
    `splits`: that many ranges of keys (1 to 8), None: by `decode_splits`."""
    k4, ks, v4, vs, pages, nkv, page_size, hd = _kv4(tensors)
    S = kv_lens.numel()
    _queries(q, nh, nkv, hd, S)
    if not decode_supported(q, hd, scale):
        raise ops.KernelError("attention_kv4_decode: bfloat16, heads of 64 or 128, rows of q on 16 bytes, a scale above 0")
    _i32(kv_lens, "kv_lens", S)
    _table(block_table, S)
    G = nh // nkv
    if splits is None:
        seen = min(max_kv_len, window) if window else max_kv_len
        splits = decode_splits(S, nkv * (-(-G // 8) if G <= 8 else -(-G // 16)), seen, sm100.init(q.device).sm_count, hd)
    if out is None:
        out = torch.empty((S, nh * hd), dtype=q.dtype, device=q.device)
    ops._check(ops._fn("quant", "rllm_kv4_decode")(
        q.data_ptr(), q.stride(0), k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, out.data_ptr(), out.stride(0),
        kv_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), S, nh, nkv, hd, page_size, float(scale), int(window or 0),
        int(splits), ops._stream()), "attention_kv4_decode")
    return out


def _runs(ctx) -> list:
    """The step's sequences as runs of neighbours that bring one token each, or more: [(first, last + 1, first row, last row + 1, single,
    longest portion, most keys)]. Worked out once a forward pass."""
    runs = ctx.per_forward.get("kv4_runs")
    if runs is None:
        runs, row = [], 0
        keys = ctx.kv_lens_host or [ctx.max_kv_len] * ctx.num_seqs
        for s, (n, kv) in enumerate(zip(ctx.q_lens_host, keys)):
            if runs and runs[-1][4] == (n == 1):
                a, _, r, _, one, longest, most = runs[-1]
                runs[-1] = (a, s + 1, r, row + n, one, max(longest, n), max(most, kv))
            else:
                runs.append((s, s + 1, row, row + n, n == 1, n, kv))
            row += n
        ctx.per_forward["kv4_runs"] = runs
    return runs


def _portions(q, tensors, ctx, block_table, nh, scale, window, run, out, scratch) -> bool:
    """Attention of a run of portions (bfloat16, heads of 64 or 128): the keys and values that they see are read into scratch, in pages of
    READ_PAGE places, and the kernels of the cache of whole numbers attend over those. A portion's rows share the keys, so the
    numbers are made once instead of in every row tile. Keys are rounded to bfloat16, what the queries' product takes; values (12
    significant bits) and the weights that meet them to half precision with a power of two a page: with both in bfloat16 the result was
    0.0026 of its norm from the exact one, with half precision 0.0018, of which 0.0017 is the output's own rounding. False where the
    memory left does not hold the scratch."""
    s0, s1, r0, r1, _, longest, most = run
    k4, ks, v4, vs, pages, nkv, page_size, hd = _kv4(tensors)
    S, width, T = s1 - s0, -(-most // READ_PAGE), r1 - r0
    size = S * width * nkv * READ_PAGE * hd * 2
    if S > 1 and 2 * size > READ_BYTES:            # one by one, then
        row = r0
        for s in range(s0, s1):
            n = ctx.q_lens_host[s]
            if not _portions(q, tensors, ctx, block_table, nh, scale, window, (s, s + 1, row, row + n, False, n, ctx.kv_lens_host[s]), out, scratch):
                return False
            row += n
        return True
    room = scratch(2 * size, lambda: torch.empty((2, S * width, nkv, READ_PAGE, hd), dtype=torch.bfloat16, device=q.device))
    if room is None:
        return False
    k, v = room[0], room[1].view(torch.float16)
    meta = torch.empty(S * width * (1 + nkv) + S + 1, dtype=torch.int32, device=q.device)
    table, vexp, cu = meta[: S * width].view(S, width), meta[S * width: S * width * (1 + nkv)], meta[S * width * (1 + nkv):]
    kv_lens, bt = ctx.kv_lens[s0:s1], block_table[s0:s1]
    ops._check(ops._fn("quant", "rllm_kv4_read")(
        ops.DT_BF16, k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, bt.data_ptr(), bt.stride(0), kv_lens.data_ptr(),
        ctx.cu_q[s0:].data_ptr(), int(window or 0), S, width, READ_PAGE, k.data_ptr(), v.data_ptr(), table.data_ptr(),
        cu.data_ptr(), vexp.data_ptr(), nkv, page_size, hd, ops._stream()), "kv4_read")
    a = (q[r0:r1], k, v, cu, kv_lens, table)
    if longest * (nh // nkv) >= 128 and most >= sm100.TC_ATTENTION_MIN_KEYS and sm100.prefill_tc_supported(a[0], k):
        sm100.attention_prefill_tc(*a, longest, nh, scale, window, out=out[r0:r1], vexp=vexp)
    else:
        sm100.attention_fa(*a, T, longest, most, nh, scale, window, out=out[r0:r1], vexp=vexp)
    return True


def attention_kv4(q: torch.Tensor, tensors: dict, ctx, block_table: torch.Tensor, nh: int, scale: float, window: int | None,
                  fast: bool, scratch) -> torch.Tensor:
    """A step's attention over keys and values held in 4 bits: single tokens and portions each in their kernel on the tensor cores
    (`fast`), all else on the CUDA cores. `scratch(bytes, make)`: make(), or None where the memory left does not hold it."""
    hd = 2 * tensors["k4"].shape[3]
    simt = lambda: attention_kv4_simt(q, tensors, ctx.token_seq, ctx.positions, block_table, nh, scale, window)
    if not fast or not decode_supported(q, hd, scale):
        return simt()
    if ctx.max_q_len == 1:
        return attention_kv4_decode(q, tensors, ctx.kv_lens, block_table, nh, scale, window, ctx.max_kv_len)
    _queries(q, nh, tensors["k4"].shape[1], hd, ctx.num_tokens)
    out = torch.empty((q.shape[0], nh * hd), dtype=q.dtype, device=q.device)
    for run in _runs(ctx):
        s0, s1, r0, r1, single, _, most = run
        if single:
            attention_kv4_decode(q[r0:r1], tensors, ctx.kv_lens[s0:s1], block_table[s0:s1], nh, scale, window, most, out=out[r0:r1])
        elif not _portions(q, tensors, ctx, block_table, nh, scale, window, run, out, scratch):
            return simt()
    return out
