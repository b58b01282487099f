"""Python face of the kernels of quantised serving (library "quant"): rows and weights in 8 bits with a scale each, their
product, and keys and values held in 4 bits with the attention that reads them.

A row in 8 bits: scale = float32(max |x| / 127), codes x / scale to the nearest integer, ties to even. A row of zeros has a
scale of 0; one with an infinity or a NaN has a scale of NaN, and so are its products. A group of 32 numbers of a head in 4
bits: m the number of largest magnitude (the positive one of two), d = bfloat16(m / -8), codes x / d to the nearest integer, ties to
even, clamped to -8..7; the number stands for code * d. (The layout is in csrc/quant.cuh.)
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from functools import lru_cache

import torch

from . import ops, sm100

_P = c_void_p
ops.register_signatures("quant", {
    "rllm_quantize_rows": [c_int, _P, c_longlong, _P, _P, c_int, c_float, _P, c_longlong, _P, c_int, c_int, c_int, _P],
    "rllm_int8_gemm": [c_int, c_int, _P, _P, _P, _P, _P, c_longlong, c_int, c_int, c_int, c_int, _P, c_int, _P],
    "rllm_int8_plan": [c_int, c_int, c_int, c_int, c_int, _P, _P],
    "rllm_int8_linear": [c_int, c_int, c_int, _P, c_longlong, _P, _P, c_int, c_float, _P, _P, _P, _P, _P, c_longlong, c_int, c_int, c_int,
                         c_int, c_int, _P, c_int, _P],
    "rllm_kv4_store": [c_int, _P, _P, c_longlong, c_longlong, _P, _P, _P, _P, _P, c_longlong, c_int, c_int, c_int, c_int, _P],
    "rllm_kv4_read": [c_int, _P, _P, _P, _P, c_longlong, _P, c_int, _P, _P, c_int, c_int, c_int, c_int, _P, _P, c_int, _P, _P, _P, _P,
                      c_int, c_int, c_int, _P],
    "rllm_kv4_decode": [_P, c_int, _P, _P, _P, _P, c_longlong, _P, c_int, _P, _P, c_int, c_int, c_int, c_int, c_int, c_int, c_float, c_int,
                        c_int, c_int, _P],
    "rllm_kv4_attention_simt": [c_int, _P, c_int, _P, _P, _P, _P, c_longlong, _P, c_int, _P, _P, _P, c_int, c_int, c_int, c_int, c_int,
                                c_int, c_float, c_int, _P],
})

INT8_MAX_K = 131072           # 127^2 K stays below 2^31
HEAD_SIZES = (64, 128, 192, 256)


def _here(t: torch.Tensor, name: str) -> None:
    """The launch goes to the current device's current stream: a tensor of another device would be read from there."""
    d = t.get_device()                                     # -1: the CPU
    if d < 0 or d != ops._raw_device():
        ops._cuda(t, name)
        raise ops.KernelError(f"{name} is on {t.device}, the current device is cuda:{ops._raw_device()}")


class Int8Rows:
    """Rows in 8 bits: `codes` int8 [rows, width rounded up to a multiple of 16] (zeros behind the width), `scales` float32
    [rows]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, width: int):
        width = int(width)
        if (codes.dtype != torch.int8 or codes.dim() != 2 or not codes.is_contiguous() or width < 1 or codes.shape[1] != (width + 15) // 16 * 16
                or scales.dtype != torch.float32 or scales.shape != codes.shape[:1] or not scales.is_contiguous()
                or scales.device != codes.device):
            raise ops.KernelError(f"rows in 8 bits: codes must be contiguous int8 [rows, {width} rounded up to a multiple of 16], scales "
                                  "contiguous float32 [rows] beside them")
        self.codes, self.scales, self.width = codes, scales, width

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
    """A weight [N, K] in 8 bits, a scale per output channel: the backend's products take it where they take a tensor. A product copies the codes
    of a `settled` matrix before the kernel in front of it has ended; those of any other, one put together from tensors or written
    to since, only then."""
    _settled = None

    def settle(self) -> "Int8Matrix":
        """Waits for the work that writes the codes; they are not to be written after. (Nothing is waited for, and the matrix is not settled,
        while a graph is captured.)"""
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(self.device).synchronize()
            self._settled = self._version()
        return self

    def _version(self):
        return -1 if self.codes.is_inference() else self.codes._version       # (what torch counts a tensor's writes by)

    @property
    def settled(self) -> bool:
        n = self._settled
        return n is not None and (n == -1 or n == self.codes._version)


def _rows(x: torch.Tensor, norm: tuple | None, rows: torch.Tensor | None):
    """(dtype, rows, columns, norm weight or None, its dtype, eps) of rows to be quantised, checked."""
    _here(x, "x")
    dt = ops._dt(x, "x")
    if x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ops.KernelError("rows in 8 bits: x must be [T, K] with unit inner stride")
    T, K = x.shape
    if K < 1:
        raise ops.KernelError("rows in 8 bits: rows without numbers")
    if rows is not None:
        _here(rows, "rows")
        if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous():
            raise ops.KernelError("rows in 8 bits: rows must be a contiguous int32 vector")
        T = rows.numel()
    if norm is None:
        return dt, T, K, None, 0, 0.0
    w, eps = norm
    _here(w, "norm weight")
    if w.shape != (K,) or not w.is_contiguous():
        raise ops.KernelError(f"norm weight must be a contiguous [{K}], got {tuple(w.shape)}")
    return dt, T, K, w.data_ptr(), ops._dt(w, "norm weight"), eps


def quantize_rows(x: torch.Tensor, norm: tuple | None = None, rows: torch.Tensor | None = None, cls=Int8Rows) -> Int8Rows:
    """Rows of x [T, K] (float32 or bfloat16, unit inner stride) in 8 bits. `norm` (weight, eps): of their RMSNorm, which is not
    rounded in between. `rows` int32 [R]: of those rows only."""
    dt, T, K, g, g_dt, eps = _rows(x, norm, rows)
    codes = torch.empty((T, (K + 15) // 16 * 16), dtype=torch.int8, device=x.device)
    scales = torch.empty(T, dtype=torch.float32, device=x.device)
    ops._check(ops._fn("quant", "rllm_quantize_rows")(
        dt, x.data_ptr(), x.stride(0), ops._ptr(rows), g, g_dt, float(eps), codes.data_ptr(), codes.stride(0), scales.data_ptr(), T, K,
        int(cls is Int8Rows), ops._stream()), "quantize_rows")
    return cls(codes, scales, K)


def quantize_matrix(w: torch.Tensor) -> Int8Matrix:
    """A weight [N, K] in 8 bits, a scale per row (output channel). Done when it returns (`Int8Matrix.settle`)."""
    return quantize_rows(w, cls=Int8Matrix).settle()


def _output(T: int, K: int, w: Int8Matrix, epilogue: int, out: torch.Tensor | None, out_dtype: torch.dtype, device):
    """(outputs, output tensor) of a product with w, checked."""
    if not isinstance(w, Int8Matrix):
        raise ops.KernelError("a product in 8 bits takes an Int8Matrix")
    _here(w.codes, "w")
    N = w.codes.shape[0]
    if w.width != K:
        raise ops.KernelError(f"product in 8 bits: x has {K} columns, w has {w.width}")
    if K > INT8_MAX_K:
        raise ops.KernelError(f"product in 8 bits: {K} columns; the sums are exact in 32 bits up to {INT8_MAX_K}")
    if epilogue == ops.EPI_SWIGLU:
        if N % 2:
            raise ops.KernelError("product in 8 bits: a gate/up pair has an even number of rows")
        N //= 2
    elif epilogue in (ops.EPI_STORE_F32, ops.EPI_ACCUM_F32):
        out_dtype = torch.float32
    elif epilogue != ops.EPI_STORE:
        raise ops.KernelError(f"product in 8 bits: no epilogue {epilogue}")
    if out is None:
        if epilogue == ops.EPI_ACCUM_F32:
            raise ops.KernelError("product in 8 bits: nothing to add into (`out`)")
        return N, torch.empty((T, N), dtype=out_dtype, device=device)
    _here(out, "out")
    if out.shape != (T, N) or out.dtype != out_dtype or (out.stride(1) != 1 and N > 1) or (T > 1 and out.stride(0) < N):
        raise ops.KernelError(f"product in 8 bits: out must be {out_dtype} [{T}, {N}] with unit inner stride and rows side by side")
    return N, out


def linear_int8(x: Int8Rows, w: Int8Matrix, epilogue: int = ops.EPI_STORE, out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x w^T from the codes: the integer sums are exact, times both scales in float. `epilogue`: `ops.EPI_STORE` (rounded once to
    out_dtype), `EPI_STORE_F32`, `EPI_ACCUM_F32` (added into the float `out`) or `EPI_SWIGLU` (w = [gate; up])."""
    if not isinstance(x, Int8Rows) or isinstance(x, Int8Matrix):
        raise ops.KernelError("linear_int8 takes Int8Rows (numbers: linear)")
    _here(x.codes, "x")
    T, K = x.shape
    N, out = _output(T, K, w, epilogue, out, out_dtype, x.codes.device)
    st = sm100.init(x.codes.device)
    ops._check(ops._fn("quant", "rllm_int8_gemm")(
        epilogue, ops._dt(out, "out"), x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(),
        max(out.stride(0), N), T, N, x.codes.shape[1], int(w.settled), st.err.data_ptr(), st.sm_count, ops._stream()), "linear_int8")
    return out


_NEEDS_SCRATCH = 1000000
# Tokens up to which a product may quantise them itself (int8_stream.cu has the whole rule)
STREAM_TOKENS = 8


def linear(x: torch.Tensor, w: Int8Matrix, epilogue: int = ops.EPI_STORE, out: torch.Tensor | None = None,
           out_dtype: torch.dtype = torch.bfloat16, norm: tuple | None = None, rows: torch.Tensor | None = None) -> torch.Tensor:
    """x w^T in 8 bits from numbers: `linear_int8(quantize_rows(x, norm, rows), w, ...)`, in one kernel for few tokens."""
    dt, T, K, g, g_dt, eps = _rows(x, norm, rows)
    device = x.device
    N, out = _output(T, K, w, epilogue, out, out_dtype, device)
    st = sm100.init(device)
    KP, fixed = w.codes.shape[1], int(w.settled)
    fn = ops._fn("quant", "rllm_int8_linear")
    call = lambda codes, scales: fn(
        epilogue, ops._dt(out, "out"), dt, x.data_ptr(), x.stride(0), ops._ptr(rows), g, g_dt, eps, codes, scales, w.codes.data_ptr(),
        w.scales.data_ptr(), out.data_ptr(), max(out.stride(0), N), T, N, K, KP, fixed, st.err.data_ptr(), st.sm_count, ops._stream())
    rc = call(None, None) if T <= STREAM_TOKENS else _NEEDS_SCRATCH
    launches = 1
    if rc == _NEEDS_SCRATCH:
        room = torch.empty(T * KP + 4 * T, dtype=torch.uint8, device=device)       # codes (rows of 16 bytes), then scales
        rc, launches = call(room.data_ptr(), room.data_ptr() + T * KP), 2
    ops._check(rc, "linear in 8 bits", launches)
    return out


# ---------------------------------------------------------------------------------------------
# keys and values held in 4 bits

def _kv4(tensors: dict) -> tuple:
    """(k4, ks, v4, vs, pages, kv heads, page size, head size) of a layer's tensors, checked."""
    k4, ks, v4, vs = tensors["k4"], tensors["ks"], tensors["v4"], tensors["vs"]
    shape = k4.shape
    pages, nkv, page_size, half = shape
    hd = 2 * half
    if hd not in HEAD_SIZES:
        raise ops.KernelError(f"a cache held in 4 bits has heads of {HEAD_SIZES}, not {hd}")
    here, scales = ops._raw_device(), (pages, nkv, page_size, hd // 32)
    for t, want, dt in ((k4, shape, torch.uint8), (v4, shape, torch.uint8), (ks, scales, torch.bfloat16), (vs, scales, torch.bfloat16)):
        if t.dtype != dt or t.shape != want or not t.is_contiguous() or t.get_device() != here:
            raise ops.KernelError(f"a cache held in 4 bits: codes must be contiguous uint8 {tuple(shape)} and scales bfloat16 {scales}, on the "
                                  f"current CUDA device (cuda:{here})")
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
    _here(k, "k"); _here(v, "v")
    shape = k.shape
    if len(shape) != 2 or shape[1] != nkv * hd or v.shape != shape or v.dtype != k.dtype or k.stride(1) != 1 or v.stride(1) != 1:
        raise ops.KernelError(f"kv4_store: k and v must be alike, [T, {nkv * hd}] with unit inner stride")
    T = shape[0]
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
    k, v = torch.empty((2, S, width, nkv, page_size, hd), dtype=dtype, device=k4.device).unbind(0)
    ops._check(ops._fn("quant", "rllm_kv4_read")(
        ops._dt(k, "k"), k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, block_table.data_ptr(),
        block_table.stride(0), kv_lens.data_ptr(), None, 0, S, width, page_size, k.data_ptr(), v.data_ptr(), 0, None, None, None, None, nkv, page_size, hd,
        ops._stream()), "kv4_read")
    return k, v


def _queries(q, nh, nkv, hd, T):
    _here(q, "q")
    if nh <= 0 or nh % nkv or q.dim() != 2 or q.shape[0] != T or q.shape[1] != nh * hd or q.stride(1) != 1:
        raise ops.KernelError(f"attention over 4 bits: q must be [{T}, heads * {hd}] with unit inner stride, heads a multiple of {nkv}")


def attention_kv4_simt(q: torch.Tensor, tensors: dict, token_seq: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
                       nh: int, scale: float, window: int | None = None) -> torch.Tensor:
    """Attention over 4 bits on the CUDA cores, in float: any rows, both run types, every head size. In this and every other form a visible place on
    a page that the table does not hold is a key and a value of zeros, as `kv4_read` gives it."""
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


# Places of a page in the scratch that portions are read into, and bytes of it that several sequences may take at once (more: one by one)
READ_PAGE, READ_BYTES = 128, 2 << 30


@lru_cache(maxsize=4096)
def decode_splits(base: int, keys: int, sm_count: int, hd: int) -> int:
    """Ranges the keys of a sequence are cut into (= CTAs of a cluster), `base` CTAs without: by the time in us of the rounds of CTAs over
    the places, two an SM: 2.6 before the first key (4 in later rounds), 0.0047 a key at heads of 64 and 0.007 at 128, a tenth (three tenths)
    more where two share an SM (the CTAs of a cluster of 16 do), and 1.6 + 0.1 a range for a cluster's merge."""
    best, cost = 1, None
    step, shared = (0.0047, 1.1) if hd == 64 else (0.007, 1.3)
    for s in (1, 2, 3, 4, 5, 6, 7, 8, 16):
        n = base * s
        if s > 1 and keys < 64 * s or s > 8 and n > sm_count:
            break
        rounds = -(-n // (2 * sm_count))
        if s in (3, 5, 6, 7, 8) and n > sm_count and n * 16 > rounds * 2 * sm_count * 13:    # such clusters do not fill a GPC evenly
            continue
        c = 2.6 + 4 * (rounds - 1) + rounds * step * (shared if n > sm_count or s > 8 else 1) * keys / s + (1.6 + 0.1 * s if s > 1 else 0)
        if cost is None or c < cost:
            best, cost = s, c
    return best


def decode_supported(q: torch.Tensor, hd: int, scale: float) -> bool:
    """Does the tensor-core kernel for single tokens take these queries?"""
    return q.dtype == torch.bfloat16 and hd in (64, 128) and scale > 0 and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0


def attention_kv4_decode(q: torch.Tensor, tensors: dict, kv_lens: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float,
                         window: int | None, max_kv_len: int, splits: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over 4 bits for one bfloat16 query row per sequence, heads of 64 or 128. `max_kv_len`: about how many keys a sequence has
    (for the number of ranges only); `splits`: that many ranges of keys (1 to 8, 16), None: by `decode_splits`."""
    kv = _kv4(tensors)
    S, nkv, hd = kv_lens.numel(), kv[5], kv[7]
    _queries(q, nh, nkv, hd, S)
    if not decode_supported(q, hd, scale):
        raise ops.KernelError("attention_kv4_decode: bfloat16, heads of 64 or 128, rows of q on 16 bytes, a scale above 0")
    if splits is not None and splits not in (1, 2, 3, 4, 5, 6, 7, 8, 16):
        raise ops.KernelError(f"attention_kv4_decode: 1 to 8 or 16 ranges of keys, not {splits}")
    _i32(kv_lens, "kv_lens", S)
    _table(block_table, S)
    if out is None:
        out = q.new_empty((S, nh * hd))
    else:
        _here(out, "out")
        if out.shape != q.shape or out.dtype != q.dtype or out.stride(1) != 1 or (S > 1 and out.stride(0) < nh * hd):
            raise ops.KernelError(f"attention_kv4_decode: out must be bfloat16 [{S}, {nh * hd}] with unit inner stride and rows side by side")
    _decode(q, kv, kv_lens, block_table, nh, scale, window, max_kv_len, splits, out, 0, 0, S)
    return out


def _decode(q, kv, kv_lens, block_table, nh, scale, window, max_kv_len, splits, out, row, seq, S) -> None:
    """The launch, for S sequences from `seq` on, whose rows of q and out begin at `row` (views of them would cost as much as the launch)."""
    k4, ks, v4, vs, pages, nkv, page_size, hd = kv
    sms = sm100.init(q.device).sm_count
    if splits is None:
        seen = min(max_kv_len, window) if window else max_kv_len
        splits = decode_splits(S * nkv * -(-(nh // nkv) // 16), seen, sms, hd)
    q_ld, out_ld, bt_ld = q.stride(0), out.stride(0), block_table.stride(0)
    ops._check(ops._fn("quant", "rllm_kv4_decode")(
        q.data_ptr() + 2 * row * q_ld, q_ld, k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, out.data_ptr() + 2 * row * out_ld,
        out_ld, kv_lens.data_ptr() + 4 * seq, block_table.data_ptr() + 4 * seq * bt_ld, bt_ld, S, nh, nkv, hd, page_size, float(scale),
        int(window or 0), int(splits), sms, ops._stream()), "attention_kv4_decode")


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


def portion_parts(items: int, keys: int, hd: int, sm_count: int) -> int:
    """CTAs that share a work item's keys (256 rows of a kv head, 1, 2 or 4 CTAs) where the items leave SMs idle: by the time in us, 0.0139 a
    key at heads of 64 and 0.0185 at 128, and 4 + 1/16 a CTA for where the ranges meet, 4 more for many clusters of 4. One | two | four, us with the
    keys' reading: 512 rows over 2,012 keys (32 / 8 heads of 128) 51 | 42; 512 over 600 24.6 | 27.6; 128 over 4,000 84 | 57 | 41; 64 over
    4,000 (heads of 64) 65 | 42 | 30; 512 over 8,000 116 | 71."""
    best, cost = 1, keys * (0.0139 if hd == 64 else 0.0185)
    for z in (2, 4):
        n = items * z
        c = keys * (0.0139 if hd == 64 else 0.0185) / z + 4 + n / 16 + (4 if z == 4 and n > 64 else 0)
        if n <= sm_count and c < cost:
            best, cost = z, c
    return best


def _portions(q, kv, ctx, block_table, nh, scale, window, run, out, scratch) -> bool:
    """Attention of a run of portions (bfloat16, heads of 64 or 128): the keys and values that they see are read into scratch, in pages of
    READ_PAGE places, and the kernels of the cache of whole numbers attend over those. A portion's rows share the keys, so the
    numbers are made once instead of in every row tile. Keys are rounded to bfloat16, what the queries' product takes (single tokens
    multiply the codes, which is exact); values (12 significant bits) and the weights that meet them to half precision with a power of two a
    page, or to bfloat16 on a page whose scales are too far apart for that (kv4_cache.cu): with both in bfloat16 the result was 0.0026 of
    its norm from the exact one, with half precision 0.0018, of which 0.0017 is the output's own rounding. False where the memory left does
    not hold the scratch."""
    s0, s1, r0, r1, _, longest, most = run
    k4, ks, v4, vs, pages, nkv, page_size, hd = kv
    S, T, entries = s1 - s0, r1 - r0, -(-most // READ_PAGE)
    # pages of a sequence that its rows see any place of: `span` places, wherever in a page they begin
    span = window + longest - 1 if window else most
    width = min(entries, (span + READ_PAGE - 2) // READ_PAGE + 1)
    size = S * width * nkv * READ_PAGE * hd * 2
    if S > 1 and 2 * size > READ_BYTES:            # one by one, then
        row = r0
        for s in range(s0, s1):
            n = ctx.q_lens_host[s]
            keys = ctx.kv_lens_host[s] if ctx.kv_lens_host else most
            if not _portions(q, kv, ctx, block_table, nh, scale, window, (s, s + 1, row, row + n, False, n, keys), out, scratch):
                return False
            row += n
        return True
    room = scratch(2 * size, lambda: torch.empty((2, S * width, nkv, READ_PAGE, hd), dtype=torch.bfloat16, device=q.device))
    if room is None:
        return False
    k, v = room.unbind(0)
    v = v.view(torch.float16)
    heads = S * width * nkv
    lost = heads * (hd // 32) * (READ_PAGE // 32)
    table, vexp, vlost, cu = q.new_empty(S * entries + heads + lost + S + 1, dtype=torch.int32).split((S * entries, heads, lost, S + 1))
    whole = S == ctx.num_seqs                      # (a view costs the host as much as half a launch)
    kv_lens = ctx.kv_lens if whole else ctx.kv_lens[s0:s1]
    if not whole:
        q, out = q[r0:r1], out[r0:r1]
    ops._check(ops._fn("quant", "rllm_kv4_read")(
        ops.DT_BF16, k4.data_ptr(), ks.data_ptr(), v4.data_ptr(), vs.data_ptr(), pages, block_table.data_ptr() + 4 * s0 * block_table.stride(0),
        block_table.stride(0), kv_lens.data_ptr(), ctx.cu_q.data_ptr() + 4 * s0, int(window or 0), S, width, READ_PAGE, k.data_ptr(), v.data_ptr(), entries, table.data_ptr(),
        cu.data_ptr(), vexp.data_ptr(), vlost.data_ptr(), nkv, page_size, hd, ops._stream()), "kv4_read")
    a = (q, k, v, cu, kv_lens, table.view(S, entries))
    if longest * (nh // nkv) >= 128 and most >= sm100.TC_ATTENTION_MIN_KEYS and sm100.prefill_tc_supported(q, k):
        items = -(-longest * (nh // nkv) // 256) * nkv * S
        parts = portion_parts(items, min(most, window + longest) if window else most, hd, sm100.init(q.device).sm_count)
        sm100.attention_prefill_tc(*a, longest, nh, scale, window, out=out, vexp=vexp, vlost=vlost, parts=parts)
    else:
        sm100.attention_fa(*a, T, longest, most, nh, scale, window, out=out, vexp=vexp, vlost=vlost)
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
        # a captured step's bound serves contexts from half of it up
        keys = ctx.max_kv_len * 3 // 4 if ctx.graph_safe else ctx.max_kv_len
        return attention_kv4_decode(q, tensors, ctx.kv_lens, block_table, nh, scale, window, max(keys, 1))
    kv = _kv4(tensors)
    _queries(q, nh, kv[5], hd, ctx.num_tokens)
    _i32(ctx.kv_lens, "kv_lens", ctx.num_seqs)
    _table(block_table, ctx.num_seqs)
    out = q.new_empty((q.shape[0], nh * hd))
    for run in _runs(ctx):
        s0, s1, r0, r1, single, _, most = run
        if single:
            _decode(q, kv, ctx.kv_lens, block_table, nh, scale, window, most, None, out, r0, s0, s1 - s0)
        elif not _portions(q, kv, ctx, block_table, nh, scale, window, run, out, scratch):
            return simt()
    return out
