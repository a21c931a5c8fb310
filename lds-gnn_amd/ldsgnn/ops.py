"""Torch-facing hot-path ops over the C-ABI library, with autograd.

Graphs never exist as dense N×N matrices here.  A sampled graph is a
`SampledGraph`: the symmetric bit matrix + CSR (self-loops included) +
s = deg^-1/2 on device, plus a back-link to θ for the hypergradient.

Gradients w.r.t. θ are low-rank.  Each aggregation Y = ÂZ of a graph
contributes dL/dÂ = G Zᵀ (G = dL/dY), and the θ-gradient of the whole graph is
a rank-2k symmetric update of the packed triangle (lds_theta_grad).  To get
there through PyTorch autograd — including the create_graph inner steps and
the double backward of the hyper step — every graph carries a small "token"
tensor (n × width, produced from θ by _GraphToken).  Each aggregation that
uses the graph reserves its own columns ("slot") of the token; its backward
returns the slot factors [s⊙G | s⊙Z | r] in those columns and zeros elsewhere,
so autograd's sum over uses concatenates the factors.  _GraphToken.backward
then assembles dθ once per graph.  A is differentiated once, so the factors
never need their own gradient ("closure of the kernel set").
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import numpy as np
import torch
from torch.autograd import Function, forward_ad

from . import _native as nat
from .rng import TAG_DROP_H, TAG_DROP_X, Generator, default_generator

_FULL_CAPACITY_LIMIT = 1 << 26  # col buffer upper bound n*n below this many entries

TOKEN_KCAP = 64  # U and V columns per token chunk (4 slots of 16 features)
TOKEN_RCAP = 8   # r columns per token chunk


def _stream(t: torch.Tensor) -> int:
    return nat.stream_of(t.device)


def _f32c(t: torch.Tensor, what: str) -> torch.Tensor:
    nat.require_device(t, what)
    if t.dtype != torch.float32:
        raise TypeError(f"ldsgnn {what}: expected float32, got {t.dtype}")
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.size(1):
        return t
    return t.contiguous()


def _no_tangent(what: str, *tensors) -> None:
    """Forward-mode derivatives are not implemented: a tangent is refused, where
    the direct launch would drop it."""
    if forward_ad._current_level < 0:
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"ldsgnn {what}: no forward-mode derivative; use reverse mode")


# ---------------------------------------------------------------------------
# graph containers
# ---------------------------------------------------------------------------


class CsrGraph:
    """A normalised graph on device: Â = diag(s)·Ã·diag(s) in CSR form.

    `row_ptr` (n+1, int32), `col` (>= nnz, int32, ascending per row, self-loop
    included), `s` (n, fp32), `deg` (n, int32), optional `bits` (n × words
    uint64 stored as int64) — the layouts of include/ldsgnn.h.
    """

    # columns ascending and distinct in [0, n) by construction (set by the
    # library's own samplers / fills; a caller-built CSR is checked)
    canonical_columns = False

    def __init__(self, n: int, row_ptr: torch.Tensor, col: torch.Tensor, s: torch.Tensor,
                 deg: torch.Tensor, bits: Optional[torch.Tensor] = None):
        self.n = n
        self.row_ptr, self.col, self.s, self.deg, self.bits = row_ptr, col, s, deg, bits
        self._nnz: Optional[int] = None

    # tensor-like surface used by the reference API (is_square_matrix etc.)
    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.n, self.n))

    def size(self, dim: Optional[int] = None):
        return self.shape if dim is None else self.n

    def dim(self) -> int:
        return 2

    @property
    def device(self) -> torch.device:
        return self.row_ptr.device

    @property
    def requires_grad(self) -> bool:
        return False

    def nnz(self) -> int:
        """Stored entries incl. self-loops (host sync on first call)."""
        if self._nnz is None:
            self._nnz = int(self.row_ptr[self.n].item())
        return self._nnz

    def num_edges(self) -> int:
        """Undirected off-diagonal edges."""
        return (self.nnz() - self.n) // 2

    # mean entries per row from which the column-blocked LDS kernel
    # (lds_spmm_norm_blocked) replaces the row-group kernel (F = 16 only)
    LONG_ROW_DEGREE = 256

    def long_rows(self) -> bool:
        return self.n >= 1024 and self.nnz() >= self.LONG_ROW_DEGREE * self.n

    def _block_ptr(self) -> torch.Tensor:
        bp = getattr(self, "_bptr", None)
        if bp is None:
            nb = nat.lib.lds_spmm_block_count(self.n)
            bp = torch.empty(self.n * (nb + 1), dtype=torch.int32, device=self.device)
            nat.call("lds_csr_block_ptr", nat.ptr(self.row_ptr), nat.ptr(self.col), self.n, nat.ptr(bp),
                     _stream(self.s))
            self._bptr = bp
        return bp

    def spmm(self, z: torch.Tensor, out: Optional[torch.Tensor] = None, beta: int = 0,
             blocked: Optional[bool] = None) -> torch.Tensor:
        """Y = Â·Z; no autograd.  Row-group kernel (lds_spmm_norm), or for long
        rows at F = 16 the CSR spill-pass kernel on the int8 matrix cores
        (lds_spmm_norm_dense; 165-168 against 414 µs for the column-blocked kernel
        at BASELINE config 5; needs the ascending columns this class holds: a
        CSR whose column order the kernel cannot aggregate faithfully raises
        ldsgnn._native.DeviceError on the graph's first call).  `blocked=True` forces the column-blocked kernel
        (lds_spmm_norm_blocked), `blocked=False` the row-group kernel."""
        z = _f32c(z, "spmm")
        if z.dim() != 2 or z.size(0) != self.n:
            raise ValueError(f"spmm: Z must be {self.n}×F, got {tuple(z.shape)}")
        f = z.size(1)
        if out is None:
            out = torch.empty((self.n, f), dtype=torch.float32, device=z.device)
        if blocked is None and f == 16 and self.long_rows() and self.n <= nat.lib.lds_spmm_dense_max_n() \
                and self.col.data_ptr() % 16 == 0:
            ws = getattr(self, "_dense_ws", None)
            if ws is None:
                ws = torch.empty(int(nat.lib.lds_spmm_dense_ws_bytes(self.n)), dtype=torch.uint8, device=z.device)
                self._dense_ws = ws
                self._dense_err = torch.zeros(1, dtype=torch.int32, device=z.device)
            # a graph this library sampled has canonical columns (the unchecked
            # form); any other CSR runs the checked form, which flags a column
            # order it cannot aggregate faithfully (a property of the CSR:
            # read on the graph's first call, one sync)
            checked = not self.canonical_columns
            if checked and not getattr(self, "_dense_checked", False) and torch.cuda.is_current_stream_capturing():
                # the check's error word is read on the host; inside a capture it
                # never would be, so a wrong column order would give wrong sums
                # silently on every replay: verify eagerly first
                raise RuntimeError("CsrGraph.spmm: the column order of this CSR has not been checked yet; run one "
                                   "eager spmm on it before capturing (canonical_columns=False graphs are checked "
                                   "once, on the host)")
            nat.call("lds_spmm_norm_dense", nat.ptr(self.row_ptr), nat.ptr(self.col), nat.ptr(self.s), self.n,
                     nat.ptr(z), z.stride(0), nat.ptr(out), out.stride(0), beta, nat.ptr(ws), 0, 1,
                     nat.ptr(self._dense_err) if checked else 0, _stream(z))
            if checked and not getattr(self, "_dense_checked", False) and \
                    not torch.cuda.is_current_stream_capturing():
                word = int(self._dense_err.item())
                if word:
                    self._dense_err.zero_()
                    nat.raise_device_error(word, "CsrGraph.spmm (lds_spmm_norm_dense)")
                self._dense_checked = True
            return out
        use_blocked = (f == 16 and self.long_rows()) if blocked is None else blocked
        if use_blocked:
            if f != 16 or z.stride(0) % 4 or z.data_ptr() % 16:
                raise ValueError("blocked spmm: F = 16, 16-byte aligned rows")
            nb = nat.lib.lds_spmm_block_count(self.n)
            part = torch.empty((nb, self.n, 16), dtype=torch.float32, device=z.device)
            nat.call("lds_spmm_norm_blocked", nat.ptr(self._block_ptr()), nat.ptr(self.col), nat.ptr(self.s),
                     self.n, nat.ptr(z), z.stride(0), nat.ptr(out), out.stride(0), beta, nat.ptr(part), _stream(z))
            return out
        nat.call("lds_spmm_norm", nat.ptr(self.row_ptr), nat.ptr(self.col), nat.ptr(self.s), self.n,
                 nat.ptr(z), f, z.stride(0), nat.ptr(out), out.stride(0), beta, _stream(z))
        return out

    def spmm_bitmask(self, z: torch.Tensor, out: Optional[torch.Tensor] = None, beta: int = 0) -> torch.Tensor:
        """Y = Â·Z from the sampled bitmask on the int8 matrix cores
        (lds_aggregate_bitmask; F = 16; dense graphs).  Needs `bits`."""
        if self.bits is None:
            raise ValueError("spmm_bitmask: this graph carries no bitmask")
        z = _f32c(z, "spmm_bitmask")
        if z.dim() != 2 or z.size(0) != self.n or z.size(1) != 16:
            raise ValueError(f"spmm_bitmask: Z must be {self.n}×16, got {tuple(z.shape)}")
        if out is None:
            out = torch.empty((self.n, 16), dtype=torch.float32, device=z.device)
        ws = torch.empty(int(nat.lib.lds_bitmask_agg_ws_bytes(self.n)), dtype=torch.uint8, device=z.device)
        nat.call("lds_aggregate_bitmask", nat.ptr(self.bits), self.bits.size(1), nat.ptr(self.s), self.n, nat.ptr(z),
                 z.stride(0), nat.ptr(out), out.stride(0), beta, nat.ptr(ws), _stream(z))
        return out

    def to_dense(self) -> torch.Tensor:
        """Ã as a dense 0/1 matrix (diagonal = 1).  Inspection only."""
        n = self.n
        rp = self.row_ptr.long()
        counts = rp[1:] - rp[:-1]
        rows = torch.repeat_interleave(torch.arange(n, device=self.device), counts)
        cols = self.col[: int(rp[-1].item())].long()
        a = torch.zeros((n, n), dtype=torch.float32, device=self.device)
        a[rows, cols] = 1.0
        return a

    def normalized_dense(self) -> torch.Tensor:
        """Â as a dense matrix.  Inspection only."""
        return self.s[:, None] * self.to_dense() * self.s[None, :]


class _TokenChunk:
    def __init__(self, graph: "SampledGraph", kcap: int, rcap: int):
        self.graph = graph
        self.kcap, self.rcap = kcap, rcap
        self.kused = 0
        self.rused = 0
        self.token: Optional[torch.Tensor] = None

    @property
    def width(self) -> int:
        return 2 * self.kcap + self.rcap


class SampledGraph(CsrGraph):
    """A graph drawn from θ.  Gradients flow to θ through the token chunks."""

    canonical_columns = True  # the sampler's fill writes each row's columns ascending

    def __init__(self, n, row_ptr, col, s, deg, bits, theta: Optional[torch.Tensor]):
        super().__init__(n, row_ptr, col, s, deg, bits)
        self.theta = theta
        self._chunks: List[_TokenChunk] = []

    @property
    def requires_grad(self) -> bool:
        return self.theta is not None and self.theta.requires_grad and torch.is_grad_enabled()

    def new_slot(self, f: int) -> Tuple[Optional[torch.Tensor], Optional[Tuple[int, int]]]:
        """Reserve f U/V columns + 1 r column for one aggregation."""
        if not self.requires_grad:
            return None, None
        fpad = (f + 3) & ~3
        ch = self._chunks[-1] if self._chunks else None
        if ch is None or ch.kused + fpad > ch.kcap or ch.rused + 1 > ch.rcap:
            ch = _TokenChunk(self, max(TOKEN_KCAP, fpad), TOKEN_RCAP)
            ch.token = _GraphToken.apply(self.theta, ch)
            self._chunks.append(ch)
        slot = (ch.kused, ch.rused)
        ch.kused += fpad
        ch.rused += 1
        return ch.token, (id(ch), slot[0], slot[1], fpad, ch)


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------


def sample_graph_from_triu(theta: torch.Tensor, n: int, generator: Optional[Generator] = None,
                           u_inject: Optional[torch.Tensor] = None, track_grad: bool = True,
                           keep: Optional[torch.Tensor] = None) -> SampledGraph:
    """Draw A ~ Bernoulli(clamp(θ, 0, 1)) on the upper triangle, symmetrise, add
    self-loops, build CSR + s (lds_sample_graph).  `u_inject`: n×n uniforms
    replacing the keyed Philox draws (reference-RNG parity mode).  `keep`
    (packed triu, 0/1): sparsification of the SAMPLE (src/models/sampling.py:
    19-44 applied to the Bernoulli draw) — entry (i, j) is drawn as
    u_ij < θ_ij·keep_ij, i.e. exactly sample ⊙ keep with the same uniforms,
    while the straight-through gradient still reaches every θ_ij."""
    nat.require_device(theta, "sample")
    if theta.dim() != 1 or theta.numel() != n * (n + 1) // 2 or theta.dtype != torch.float32:
        raise ValueError("theta must be the float32 packed upper triangle incl. diagonal")
    th = theta.detach()
    if not th.is_contiguous():
        th = th.contiguous()
    if keep is not None:
        if keep.shape != th.shape:
            raise ValueError("keep must be a packed upper-triangle mask like theta")
        th = (th.clamp(0.0, 1.0) * (keep.detach().to(th.device) != 0).to(th.dtype)).contiguous()
    gen = generator or default_generator
    seed, tag, counter = gen.next_graph()
    dev = theta.device
    words = nat.lib.lds_bitmask_words(n)
    bits = torch.empty((n, words), dtype=torch.int64, device=dev)
    deg = torch.empty(n, dtype=torch.int32, device=dev)
    row_ptr = torch.empty(n + 1, dtype=torch.int32, device=dev)
    s = torch.empty(n, dtype=torch.float32, device=dev)
    st = _stream(th)
    if u_inject is not None:
        u_inject = _f32c(u_inject, "sample u_inject")
        if u_inject.shape != (n, n) or not u_inject.is_contiguous():
            raise ValueError("u_inject must be a contiguous n×n float32 tensor")
    nat.call("lds_sample_bitmask", nat.ptr(th), n, seed, tag, counter, nat.ptr(u_inject),
             nat.ptr(bits), words, st)
    nat.call("lds_bitmask_degree", nat.ptr(bits), n, words, nat.ptr(deg), nat.ptr(s), st)
    nat.call("lds_exclusive_scan", nat.ptr(deg), n, nat.ptr(row_ptr), st)
    if n * n <= _FULL_CAPACITY_LIMIT:
        capacity = n * n
    else:  # exact size: one host sync
        capacity = int(row_ptr[n].item())
    col = torch.empty(max(capacity, 1), dtype=torch.int32, device=dev)
    nat.call("lds_bitmask_fill_csr", nat.ptr(bits), n, words, nat.ptr(row_ptr), nat.ptr(col),
             capacity, 0, st)
    return SampledGraph(n, row_ptr, col, s, deg, bits, theta if track_grad else None)


def csr_graph_from_dense(adj: torch.Tensor) -> CsrGraph:
    """A fixed 0/1 adjacency (e.g. the dataset graph) in the
    hot-path layout.  Off-diagonal entries must be 0/1 and symmetric; the
    diagonal is ignored (self-loops are set, src/utils/graph.py:123-133)."""
    nat.require_device(adj, "csr_graph_from_dense")
    n = adj.size(0)
    a = adj.detach().to(torch.float32).clone()
    a.fill_diagonal_(1.0)
    if not bool(((a == 0) | (a == 1)).all()) or not torch.equal(a, a.t()):
        raise ValueError("csr_graph_from_dense needs a symmetric 0/1 adjacency")
    deg = a.sum(1).to(torch.int32)
    row_ptr = torch.zeros(n + 1, dtype=torch.int32, device=adj.device)
    row_ptr[1:] = torch.cumsum(deg, 0).to(torch.int32)
    col = a.nonzero()[:, 1].to(torch.int32).contiguous()  # row-major -> ascending per row
    s = torch.empty(n, dtype=torch.float32, device=adj.device)
    # same correctly-rounded reciprocal(sqrt(d)) as the sampler's degree pass
    nat.call("lds_csr_degree_scale", nat.ptr(row_ptr), n, nat.ptr(deg), nat.ptr(s), _stream(s))
    return CsrGraph(n, row_ptr, col, s, deg, None)


# ---------------------------------------------------------------------------
# autograd functions
# ---------------------------------------------------------------------------


class _GraphToken(Function):
    """θ -> zero token; backward assembles dθ of one graph (lds_theta_grad)."""

    @staticmethod
    def forward(ctx, theta, chunk):
        ctx.chunk = chunk
        ctx.theta = theta.detach()  # clamp mask read at backward time (θ stays in [0,1])
        return torch.zeros((chunk.graph.n, chunk.width), dtype=torch.float32, device=theta.device)

    @staticmethod
    def backward(ctx, dtok):
        ch: _TokenChunk = ctx.chunk
        theta = ctx.theta
        dtok = dtok.contiguous()
        grad = torch.empty_like(theta)
        w = ch.width
        base = dtok.data_ptr()
        nat.call("lds_theta_grad", base, base + 4 * ch.kcap, w, ch.kused, base + 8 * ch.kcap, w,
                 ch.rused, nat.ptr(theta), ch.graph.n, nat.ptr(grad), 0, form_code(), _stream(theta))
        return grad, None


def _write_slot(dtok: torch.Tensor, slot, gy: torch.Tensor, z: torch.Tensor, y: torch.Tensor,
                dz: torch.Tensor, s: torch.Tensor, n: int) -> None:
    _, koff, roff, fpad, ch = slot
    w = ch.width
    base = dtok.data_ptr()
    f = z.size(1)
    nat.call("lds_slot_factors", nat.ptr(gy), gy.stride(0), nat.ptr(z), z.stride(0), nat.ptr(y),
             y.stride(0), nat.ptr(dz), dz.stride(0), nat.ptr(s), n, f, fpad,
             base + 4 * koff, w, base + 4 * (ch.kcap + koff), w, base + 4 * (2 * ch.kcap + roff), w,
             _stream(dtok))


class _Aggregate(Function):
    """Y = Â·Z.  Backward: dZ = Â·G (recorded when create_graph), token slot."""

    @staticmethod
    def forward(ctx, z, token, graph, slot):
        z = _f32c(z, "aggregate")
        y = graph.spmm(z)
        ctx.graph, ctx.slot = graph, slot
        ctx.save_for_backward(z, y, token)
        return y

    @staticmethod
    def backward(ctx, gy):
        z, y, token = ctx.saved_tensors
        graph, slot = ctx.graph, ctx.slot
        need_z, need_tok = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        gy = _f32c(gy, "aggregate backward")
        dz = None
        if need_z or need_tok:
            if need_z and torch.is_grad_enabled():
                dz = aggregate(gy, graph)  # create_graph: a differentiable use of the graph
            else:
                dz = graph.spmm(gy)
        dtok = None
        if need_tok:
            dtok = torch.zeros_like(token)
            with torch.no_grad():
                _write_slot(dtok, slot, gy, z, y, dz.detach(), graph.s, graph.n)
        return (dz if need_z else None), dtok, None, None


def aggregate(z: torch.Tensor, graph: CsrGraph) -> torch.Tensor:
    """Â·Z for a hot-path graph, differentiable in Z and (sampled graphs) θ."""
    _no_tangent("aggregate", z)
    if isinstance(graph, SampledGraph) and graph.requires_grad:
        token, slot = graph.new_slot(z.size(1))
        return _Aggregate.apply(z, token, graph, slot)
    if z.requires_grad and torch.is_grad_enabled():
        return _Aggregate.apply(z, None, graph, None)
    return graph.spmm(z)


def _call_on(t: torch.Tensor, name: str, *args) -> None:
    """One entry point on `t`'s device, on that device's current stream (its
    last argument), whatever the current device is."""
    index = t.get_device()
    if index == torch._C._cuda_getDevice():
        nat.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            nat.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _element_code(t: torch.Tensor, what: str) -> int:
    nat.require_device(t, what)
    code = nat.ELEMENT_CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"ldsgnn {what}: expected float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rows_of(t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(tensor, rows, cols, row stride) of `t` as a rows × last-dimension block;
    a copy only where its strides are no such block's."""
    if t.dim() == 0:
        raise ValueError(f"ldsgnn {what}: expected at least one dimension")
    cols, n = t.size(-1), t.numel()
    if cols:
        rows = n // cols
    else:
        rows = 1
        for d in t.shape[:-1]:
            rows *= d
    if n == 0 or t.is_contiguous():
        return t, rows, cols, cols
    try:
        v = t.view(rows, cols)
    except RuntimeError:
        v = None
    if v is None or (cols > 1 and v.stride(1) != 1) or (rows > 1 and v.stride(0) < cols):
        return t.contiguous(), rows, cols, cols
    return v, rows, cols, (v.stride(0) if rows > 1 else cols)


def _keep_scale(p: float, key, what: str) -> Tuple[float, float]:
    """(1 - p, 1 / (1 - p)) in fp32, as the kernels take them."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"ldsgnn {what}: p must lie in [0, 1], got {p}")
    if p > 0.0 and key is None:
        raise ValueError(f"ldsgnn {what}: dropout needs a key (seed, tag, counter)")
    if p == 0.0:
        return 1.0, 1.0
    keep = np.float32(1.0) - np.float32(p)
    return float(keep), float(np.float32(1.0) / keep) if keep > 0 else 0.0


class _KeyedDropout(Function):
    """y = residual + mask(x).  Linear: the backward is the same mask on dy (at
    any order), and dy itself for the residual."""

    @staticmethod
    def forward(ctx, x, residual, mask):
        ctx.mask = mask
        return _dropout_raw(x, mask, residual)

    @staticmethod
    def backward(ctx, gy):
        need_x, need_residual, _ = ctx.needs_input_grad
        gx = None
        if need_x and ctx.mask[0] == 1.0:  # p = 0: every element kept, scaled by 1
            gx = gy
        elif need_x:
            gx = _KeyedDropout.apply(gy, None, ctx.mask) if torch.is_grad_enabled() else _dropout_raw(gy, ctx.mask)
        return gx, (gy if need_residual else None), None


def _dropout_raw(x: torch.Tensor, mask: tuple, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """mask: (keep, scale, seed, tag, counter), the entry point's arguments."""
    xr, rows, cols, ldx = _rows_of(x, "dropout")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    at, ldr = 0, 0
    if residual is not None:
        residual, _, _, ldr = _rows_of(residual, "dropout residual")
        at = residual.data_ptr()
    _call_on(x, "lds_dropout_add", xr.data_ptr(), ldx, at, ldr, y.data_ptr(), cols, rows, cols,
             nat.ELEMENT_CODES[x.dtype], *mask)
    return y


def keyed_dropout(x: torch.Tensor, p: float, key, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """F.dropout with a keyed mask that is never stored, with an optional
    residual added in the same pass (lds_dropout_add):
        y = residual + (u(i, j) < 1 - p ? x / (1 - p) : 0)
    x: float32, bfloat16 or float16, one or more dimensions, any strides; row i
    counts the positions of all but the last dimension, j is the position in
    it.  `residual`: shape, dtype and device of x (it is not broadcast).  The
    result is rounded once.  key: (seed, tag, counter), see
    ldsgnn.rng.Generator.dropout_key; p in [0, 1]."""
    keep, scale = _keep_scale(p, key, "dropout")
    _no_tangent("dropout", x, residual)
    _element_code(x, "dropout")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or
                                 residual.device != x.device):
        raise ValueError(f"ldsgnn dropout: the residual must match x ({tuple(x.shape)}, {x.dtype}, {x.device}), got "
                         f"{tuple(residual.shape)}, {residual.dtype}, {residual.device}")
    seed, tag, counter = key if key is not None else (0, 0, 0)
    mask = (keep, scale, seed, tag, counter)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _KeyedDropout.apply(x, residual, mask)
    return _dropout_raw(x, mask, residual)


# ---------------------------------------------------------------------------
# group norm with an activation, channels last
# ---------------------------------------------------------------------------

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}


class _NormPlan:
    """The constants of one group_norm_act call."""
    __slots__ = ("groups", "act", "eps", "keep", "mask")

    def __init__(self, groups, act, eps, keep, scale, key):
        self.groups, self.act, self.eps, self.keep = groups, act, eps, keep
        self.mask = (keep, scale, *(key if key is not None else (0, 0, 0)))


def _samples_of(t: torch.Tensor) -> Tuple[torch.Tensor, int, int, int, int]:
    """(tensor, samples, n, sample stride, row stride) of a (..., n, C) tensor;
    a copy only where its strides are no such block's."""
    n, c = t.size(-2), t.size(-1)
    samples = 1
    for d in t.shape[:-2]:
        samples *= d
    if t.is_contiguous():
        return t, samples, n, n * c, c
    if t.numel() == 0:
        return t.contiguous(), samples, n, n * c, c
    try:
        v = t.view(samples, n, c)
    except RuntimeError:
        v = None
    if v is None or (c > 1 and v.stride(2) != 1) or (n > 1 and v.stride(1) < c):
        return t.contiguous(), samples, n, n * c, c
    return v, samples, n, v.stride(0), (v.stride(1) if n > 1 else c)


def _norm_forward(x, weight, bias, pl: _NormPlan):
    code = nat.ELEMENT_CODES[x.dtype]
    xr, samples, n, sx, ldx = _samples_of(x)
    c = x.size(-1)
    dev = x.device
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = torch.empty((2, samples, pl.groups), dtype=torch.float32, device=dev)
    if x.numel() == 0:
        return y, stats
    pcode = 0 if weight is None and bias is None else nat.ELEMENT_CODES[(bias if weight is None else weight).dtype]
    size = nat.lib.lds_group_norm_ws_bytes(samples, n, c, pl.groups, code, 0)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    at = stats.data_ptr()
    _call_on(x, "lds_group_norm_forward", xr.data_ptr(), sx, ldx, samples, n, c, pl.groups, code, nat.ptr(weight),
             nat.ptr(bias), pcode, pl.eps, pl.act, *pl.mask, y.data_ptr(), at, at + 4 * samples * pl.groups,
             nat.ptr(ws))
    return y, stats


def _norm_backward(gy, x, weight, bias, stats, pl: _NormPlan, need):
    """(dx, dweight, dbias); `need`: which of them are wanted."""
    code = nat.ELEMENT_CODES[x.dtype]
    c = x.size(-1)
    dev = x.device
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    want_w, want_b = need[1] and weight is not None, need[2] and bias is not None
    if x.numel() == 0:
        return (dx, torch.zeros_like(weight) if want_w else None, torch.zeros_like(bias) if want_b else None)
    dw = torch.empty(c, dtype=torch.float32, device=dev) if want_w else None
    db = torch.empty(c, dtype=torch.float32, device=dev) if want_b else None
    xr, samples, n, sx, ldx = _samples_of(x)
    gr, _, _, sg, ldg = _samples_of(gy)
    pcode = 0 if weight is None and bias is None else nat.ELEMENT_CODES[(bias if weight is None else weight).dtype]
    size = nat.lib.lds_group_norm_ws_bytes(samples, n, c, pl.groups, code, 1)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    at = stats.data_ptr()
    _call_on(x, "lds_group_norm_backward", gr.data_ptr(), sg, ldg, xr.data_ptr(), sx, ldx, samples, n, c, pl.groups,
             code, nat.ptr(weight), nat.ptr(bias), pcode, pl.act, *pl.mask, at, at + 4 * samples * pl.groups,
             nat.ptr(dx), nat.ptr(dw), nat.ptr(db), nat.ptr(ws))
    if pcode:  # 16-bit parameters: one rounding of the fp32 sums
        dw = dw if dw is None else dw.to(weight.dtype)
        db = db if db is None else db.to(bias.dtype)
    return dx, dw, db


def _norm_composed(x, weight, bias, mask, pl: _NormPlan):
    """group_norm_act in elementary differentiable operations (fp32): what the
    second derivative is taken of."""
    c = x.size(-1)
    v = x.float().reshape(-1, x.size(-2), pl.groups, c // pl.groups)
    d = v - v.mean((1, 3), keepdim=True)
    z = (d / (d.square().mean((1, 3), keepdim=True) + pl.eps).sqrt()).reshape(x.shape)
    if weight is not None:
        z = z * weight.float()
    if bias is not None:
        z = z + bias.float()
    z = torch.relu(z) if pl.act == 1 else z * torch.sigmoid(z) if pl.act == 2 else z
    return z if mask is None else torch.where(mask > 0, z * mask, torch.zeros_like(z))


class _GroupNormAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, pl):
        y, stats = _norm_forward(x, weight, bias, pl)
        ctx.pl = pl
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():  # create_graph: the gradient is differentiated again
            return _GroupNormActGrad.apply(gy, x, weight, bias, stats, ctx.pl, need) + (None,)
        return _norm_backward(gy, x, weight, bias, stats, ctx.pl, need) + (None,)


class _GroupNormActGrad(Function):
    """The gradient as a function of (dy, x, weight, bias).  Its own gradient is
    composed from elementary operations: only the hyper step of the autograd
    path (a double backward through the inner steps) takes it."""

    @staticmethod
    def forward(ctx, gy, x, weight, bias, stats, pl, need):
        ctx.pl, ctx.need = pl, need
        ctx.save_for_backward(gy, x, weight, bias)
        return _norm_backward(gy, x, weight, bias, stats, pl, need)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *cot):
        pl, need = ctx.pl, ctx.need
        inputs = [None if t is None else t.detach().requires_grad_(True) for t in ctx.saved_tensors]
        gy, x, weight, bias = inputs
        if x.numel() == 0:  # the first order is zeros, whatever the inputs
            return tuple(None if t is None else torch.zeros_like(t) for t in inputs) + (None, None, None)
        mask = None
        if pl.keep < 1.0:
            mask = _dropout_raw(torch.ones(x.shape, dtype=torch.float32, device=x.device), pl.mask)
        with torch.enable_grad():
            y = _norm_composed(x, weight, bias, mask, pl)
            wrt = [t for t, k in zip((x, weight, bias), need) if k and t is not None]
            first = torch.autograd.grad(y, wrt, gy.float(), create_graph=True)
            given = [c for c, t, k in zip(cot, (x, weight, bias), need) if k and t is not None]
            live = [t for t in inputs if t is not None]
            second = iter(torch.autograd.grad(first, live, given, allow_unused=True))
        return tuple(None if t is None else next(second) for t in inputs) + (None, None, None)


def group_norm_act(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, act: str = "none", eps: float = 1e-5, p: float = 0.0,
                   key=None) -> torch.Tensor:
    """Group norm, an activation and keyed dropout in one operator, channels last
    (lds_group_norm_forward / _backward):
        y = mask · act((x - mean) / sqrt(var + eps) · weight + bias)
    x: (..., n, C), float32, bfloat16 or float16, any strides; every leading
    position is a sample of n nodes, normalised by itself over its nodes and
    the C / groups channels of each group (biased variance).  weight, bias: C
    values, float32, bfloat16 or float16 (both alike), or None.  act: "none",
    "relu" or "silu".  p > 0: the mask of keyed_dropout(·, p, key) on the result.
    Differentiable in x, weight and bias, twice where create_graph asks for it.
    The result is rounded once; statistics and sums are fp32."""
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"ldsgnn group_norm_act: unknown activation {act!r}; one of {sorted(ACTIVATIONS)}")
    _no_tangent("group_norm_act", x, weight, bias)
    _element_code(x, "group_norm_act")
    if x.dim() < 2:
        raise ValueError(f"ldsgnn group_norm_act: expected (..., n, C), got {tuple(x.shape)}")
    c = x.size(-1)
    if isinstance(groups, bool) or not isinstance(groups, int) or groups < 1 or c % groups:
        raise ValueError(f"ldsgnn group_norm_act: {groups!r} groups do not divide {c} channels")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"ldsgnn group_norm_act: eps must be finite and not negative, got {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (c,) or t.device != x.device or t.dtype not in nat.ELEMENT_CODES):
            raise ValueError(f"ldsgnn group_norm_act: {name} must hold {c} floating values on {x.device}, got "
                             f"{tuple(t.shape)}, {t.dtype}, {t.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("ldsgnn group_norm_act: weight and bias must share a dtype")
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    keep, scale = _keep_scale(p, key, "group_norm_act")
    pl = _NormPlan(groups, code, float(eps), keep, scale, key if keep < 1.0 else None)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _GroupNormAct.apply(x, weight, bias, pl)
    return _norm_forward(x, weight, bias, pl)[0]


# ---------------------------------------------------------------------------
# 8-bit integer product
# ---------------------------------------------------------------------------

INT8_MAX_K = 131071  # k·127·127 and k·128·128 stay below 2^31


def _int8_stride(k: int) -> int:
    """Row stride (bytes) of the 8-bit layouts: an odd number of 64-byte lines, so
    that the 16 rows a wave reads at once do not fall on the same cache sets
    (16 x 4096 x 4096: 5.9 us at stride 4096, 4.8 at 4160); short rows are only
    padded to 16 bytes."""
    return -(-k // 16) * 16 if k <= 512 else (-(-k // 64) | 1) * 64


def _int8_readable(q: torch.Tensor, what: str) -> torch.Tensor:
    """q where the product can read it (16-byte rows that end inside their
    storage), else a copy."""
    nat.require_device(q, what)
    if q.dtype != torch.int8 or q.dim() != 2:
        raise TypeError(f"ldsgnn {what}: expected a 2-d int8 tensor, got {q.dim()}-d {q.dtype}")
    m, k = q.shape
    if m == 0 or k == 0:
        return q
    ld = q.stride(0) if m > 1 else 16
    if (q.stride(1) == 1 or k == 1) and (ld >= k or m == 1) and ld % 16 == 0 and q.data_ptr() % 16 == 0 and \
            (k % 16 == 0 or
             q.untyped_storage().nbytes() - q.storage_offset() >= (m - 1) * ld + -(-k // 16) * 16):
        return q
    return _int8_layout(q)


def _int8_layout(q: torch.Tensor) -> torch.Tensor:
    out = torch.zeros((q.size(0), _int8_stride(q.size(1))), dtype=torch.int8, device=q.device)[:, :q.size(1)]
    out.copy_(q)
    return out


def int8_rows(q: torch.Tensor) -> torch.Tensor:
    """`q` (rows × k, int8) in the layout that the product reads best, the one
    quantize_rows writes: lay a layer's weights out once.  q itself where it has
    that layout; the product takes other layouts too, and copies the rows that
    it cannot read in place."""
    r = _int8_readable(q, "int8_rows")
    return r if r.size(0) <= 1 or r.size(1) == 0 or r.stride(0) == _int8_stride(r.size(1)) else _int8_layout(r)


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of the rows of x (rows × k; float32, bfloat16 or float16):
    scale = max|x| / 127 per row, q = x / scale to the nearest int8, ties to
    even (lds_quantize_rows).  A zero row gives q = 0, scale = 0; a row with an
    infinity or a NaN gives scale NaN.  For weights (out × in) the same call
    gives a scale per output channel.  No gradient."""
    _no_tangent("quantize_rows", x)
    code = _element_code(x, "quantize_rows")
    if x.dim() != 2:
        raise ValueError(f"ldsgnn quantize_rows: expected rows × k, got {tuple(x.shape)}")
    xr, _, cols, ldx = _rows_of(x.detach(), "quantize_rows")
    rows = x.size(0)
    wide = _int8_stride(cols)
    q = torch.empty((rows, wide), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call_on(x, "lds_quantize_rows", xr.data_ptr(), ldx, rows, cols, code, q.data_ptr(), wide, scale.data_ptr())
    return q[:, :cols], scale


def _no_grad_only(what: str, *tensors) -> None:
    _no_tangent(what, *tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"ldsgnn {what}: the 8-bit product has no gradient; call it under torch.no_grad()")


def _int8_weights(what: str, k: int, dev, wq, w_scale, bias, out_dtype):
    """The checks of the weights' side; (wq, w_scale, bias, n, row stride, codes)."""
    wq = _int8_readable(wq, what)
    n, kw = wq.shape
    code = nat.ELEMENT_CODES.get(out_dtype)
    if code is None:
        raise TypeError(f"ldsgnn {what}: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    if k != kw or k > INT8_MAX_K:
        raise ValueError(f"ldsgnn {what}: inner sizes {k} and {kw} must agree and not exceed {INT8_MAX_K}")
    if w_scale.shape != (n,) or w_scale.dtype != torch.float32 or w_scale.device != dev or wq.device != dev:
        raise ValueError(f"ldsgnn {what}: wq and w_scale ({n} float32 values) must lie on {dev}, got "
                         f"{tuple(w_scale.shape)}, {w_scale.dtype}, {w_scale.device}, {wq.device}")
    pcode = 0
    if bias is not None:
        pcode = nat.ELEMENT_CODES.get(bias.dtype)
        if bias.shape != (n,) or bias.device != dev or pcode is None:
            raise ValueError(f"ldsgnn {what}: bias must hold {n} floating values on {dev}, got "
                             f"{tuple(bias.shape)}, {bias.dtype}, {bias.device}")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    ldw = wq.stride(0) if n > 1 and k > 0 else _int8_stride(k)
    return wq, (w_scale if w_scale.is_contiguous() else w_scale.contiguous()), bias, n, ldw, pcode, code


def int8_matmul(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y = (xq wqᵀ) · x_scale per row · w_scale per output channel + bias
    (lds_int8_matmul): xq m × k and wq n × k int8 with their fp32 scales, as
    quantize_rows gives them; the sum is exact, y is float32, bfloat16 or
    float16, rounded once.  Rows that do not start at multiples of 16 bytes are
    copied (int8_rows lays them out once).  No gradient."""
    _no_grad_only("int8_matmul", x_scale, w_scale, bias)
    xq = _int8_readable(xq, "int8_matmul")
    m, k = xq.shape
    dev = xq.device
    if x_scale.shape != (m,) or x_scale.dtype != torch.float32 or x_scale.device != dev:
        raise ValueError(f"ldsgnn int8_matmul: x_scale must be {m} float32 values on {dev}, got "
                         f"{tuple(x_scale.shape)}, {x_scale.dtype}, {x_scale.device}")
    wq, w_scale, bias, n, ldw, pcode, code = _int8_weights("int8_matmul", k, dev, wq, w_scale, bias, out_dtype)
    x_scale = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
    y = torch.empty((m, n), dtype=out_dtype, device=dev)
    _call_on(xq, "lds_int8_matmul", xq.data_ptr(), xq.stride(0) if m > 1 and k > 0 else _int8_stride(k),
             x_scale.data_ptr(), wq.data_ptr(), ldw, w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(), pcode,
             m, n, k, y.data_ptr(), n, code)
    return y


def int8_linear(x: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (..., k) times an 8-bit weight (lds_int8_linear): the rows of x are
    quantised as quantize_rows does and multiplied as int8_matmul does.  Result
    (..., n) in x's dtype unless out_dtype names another.  No gradient."""
    _no_grad_only("int8_linear", x, w_scale, bias)
    xcode = _element_code(x, "int8_linear")
    if x.dim() < 1:
        raise ValueError("ldsgnn int8_linear: expected (..., k)")
    xr, m, k, ldx = _rows_of(x, "int8_linear")
    dev = x.device
    out_dtype = x.dtype if out_dtype is None else out_dtype
    wq, w_scale, bias, n, ldw, pcode, code = _int8_weights("int8_linear", k, dev, wq, w_scale, bias, out_dtype)
    y = torch.empty(x.shape[:-1] + (n,), dtype=out_dtype, device=dev)
    ldq = _int8_stride(k)
    ws = torch.empty(m * (ldq + 4), dtype=torch.uint8, device=dev)  # the rows, then their scales
    at = ws.data_ptr()
    _call_on(x, "lds_int8_linear", xr.data_ptr(), ldx, xcode, at, ldq, at + m * ldq, wq.data_ptr(), ldw,
             w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(), pcode, m, n, k, y.data_ptr(), n, code)
    return y


# ---------------------------------------------------------------------------
# plain kernels
# ---------------------------------------------------------------------------


def sgd_clamp_(theta: torch.Tensor, grad: torch.Tensor, lr: float) -> torch.Tensor:
    """θ = clamp(θ - lr·grad, 0, 1) in place (lds_sgd_clamp)."""
    nat.require_device(theta, "sgd_clamp")
    if not (theta.is_contiguous() and grad.is_contiguous()) or theta.numel() != grad.numel():
        raise ValueError("sgd_clamp_: contiguous θ and grad of equal size required")
    nat.call("lds_sgd_clamp", nat.ptr(theta), nat.ptr(grad), float(lr), theta.numel(), _stream(theta))
    return theta


def theta_grad(u: torch.Tensor, v: torch.Tensor, r: torch.Tensor, n: int,
               theta: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               accumulate: bool = False) -> torch.Tensor:
    """Packed-triangle θ-gradient from factors (lds_theta_grad).  u, v: n×k
    (already scaled by s), r: n×nr (summed per row)."""
    u, v = _f32c(u, "theta_grad"), _f32c(v, "theta_grad")
    if u.shape != v.shape or u.stride(0) != v.stride(0):
        raise ValueError("theta_grad: u and v must share shape and row stride")
    r = _f32c(r.reshape(n, -1), "theta_grad")
    if out is None:
        out = torch.empty(n * (n + 1) // 2, dtype=torch.float32, device=u.device)
    nat.call("lds_theta_grad", nat.ptr(u), nat.ptr(v), u.stride(0), u.size(1), nat.ptr(r),
             r.stride(0), r.size(1), nat.ptr(theta), n, nat.ptr(out), int(accumulate), form_code(), _stream(u))
    return out


THETA_GRAD_FORMS = {"fp32": 0, "bf16x3": 1, "bf16x3-t64k16": 2, "bf16x3-t64k32": 3, "bf16x3-t128": 4,
                    "bf16x3-t128-grouped": 5, "bf16x3-t64k16-grouped": 6, "bf16x3-t128-grouped-i64": 7,
                    "bf16x3-t128-pipe": 8, "bf16x3-t128-w8": 9, "bf16x3-direct": 10}


_theta_form = "bf16x3"


def theta_grad_form(form: Optional[str] = None) -> str:
    """Select the default arithmetic form of the θ-gradient assembly that this
    module's callers pass to the C-ABI (every lds_theta_grad* entry point takes
    the form per call; the library keeps no form state): "bf16x3" (default:
    fp32 operands split into three bf16 words, six bf16 MFMAs per product,
    fp32 accuracy; tile shape chosen by problem size), one pinned split-bf16
    variant (64-tiles with 16- or 32-wide k chunks, 128-tiles in plain or
    XCD-grouped order, the pipelined 128-tiles), "bf16x3-direct" (the
    direct-staged eight-wave 128-tile on pre-split planes: an LdsEngine then
    has its factor producers write the planes; entry points on fp32 operands
    run the by-shape form), or "fp32" (fp32-in MFMA).
    Returns the previous default.  An LdsEngine with its own `theta_form`
    ignores this default; HIP graphs keep the form they were captured with."""
    global _theta_form
    prev = _theta_form
    if form is not None:
        if form not in THETA_GRAD_FORMS:
            raise ValueError(f"unknown θ-grad form {form!r}; one of {sorted(THETA_GRAD_FORMS)}")
        _theta_form = form
    return prev


def form_code(form: Optional[str] = None) -> int:
    """The C-ABI `form` argument of `form` (default: theta_grad_form())."""
    return THETA_GRAD_FORMS[_theta_form if form is None else form]


def philox_uniform(seed: int, tag: int, counter: int, rows: int, cols: int,
                   device="cuda") -> torch.Tensor:
    out = torch.empty((rows, cols), dtype=torch.float32, device=device)
    nat.call("lds_philox_uniform", seed, tag, counter, rows, cols, nat.ptr(out), _stream(out))
    return out


__all__ = [
    "CsrGraph", "SampledGraph", "sample_graph_from_triu", "csr_graph_from_dense", "aggregate",
    "keyed_dropout", "group_norm_act", "ACTIVATIONS", "int8_rows", "quantize_rows", "int8_matmul", "int8_linear",
    "INT8_MAX_K", "sgd_clamp_", "theta_grad", "theta_grad_form", "form_code", "philox_uniform", "TAG_DROP_X", "TAG_DROP_H",
]
