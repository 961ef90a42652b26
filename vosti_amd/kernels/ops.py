"""Python bindings of the gfx950 kernel libraries.

``kernels_for(dtype)`` returns a ``Kernels`` object bound to the library built
for that element type.  Every method checks operand shapes, types and devices
on the host before a launch, because a kernel that reads out of bounds can take
the GPU down; there is no CPU path, and a missing or stale library is an error.
All launches go to torch's current stream.
"""
from __future__ import annotations

import ctypes
from ctypes import c_double, c_float, c_int, c_int64, c_uint64, c_void_p

import torch

from . import build

ABI_VERSION = 22
SEGMENT_KEYS = 256
ATTN_ITEM_ROWS = 128      # rows of one prompt item of paged_attention, and of any item of paged_attention8
CACHE8_DTYPE = torch.float8_e4m3fn
CACHE8_PAGES = (16, 256)  # smallest and largest page of an 8-bit cache

# The current stream without the object that torch.cuda.current_stream() makes around it (0.3 instead of 2.7 us of every call); not a public name, so the public one where torch lacks it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_NAMES = {torch.bfloat16: "bf16", torch.float32: "f32", "bfloat16": "bf16", "float32": "f32", "bf16": "bf16",
          "f32": "f32", "fp32": "f32"}


class KernelError(RuntimeError):
    pass


def dtype_name(dtype) -> str:
    try:
        return _NAMES[dtype]
    except KeyError:
        raise ValueError(f"unsupported element type {dtype!r}; use bfloat16 or float32") from None


def _sig(fn, *argtypes):
    fn.argtypes = list(argtypes)
    fn.restype = c_int
    return fn


class Kernels:
    def __init__(self, name: str):
        self.name = name
        self.dtype = _DTYPES[name]
        path = build.ensure(name)
        self.path = str(path)
        lib = ctypes.CDLL(self.path)
        lib.vk_last_error.restype = ctypes.c_char_p
        lib.vk_abi_version.restype = c_int
        lib.vk_elem_bytes.restype = c_int
        if lib.vk_abi_version() != ABI_VERSION:
            raise KernelError(f"{path} has ABI {lib.vk_abi_version()}, expected {ABI_VERSION}; rebuild it")
        if lib.vk_elem_bytes() != torch.empty((), dtype=self.dtype).element_size():
            raise KernelError(f"{path} was built for another element type")
        P, I, L, F = c_void_p, c_int, c_int64, c_float
        _sig(lib.vk_embedding, P, P, P, I, I, I, P)
        _sig(lib.vk_rmsnorm, P, P, P, I, I, I, I, L, L, F, P)
        _sig(lib.vk_add_rmsnorm, P, P, P, P, I, I, I, F, P)
        _sig(lib.vk_swiglu, P, P, I, I, P)
        _sig(lib.vk_gather_rows, P, P, P, I, I, P)
        _sig(lib.vk_cast_to_f32, P, P, L, P)
        _sig(lib.vk_cast_from_f32, P, P, L, P)
        _sig(lib.vk_rope_tables, P, P, P, I, I, P)
        _sig(lib.vk_fill_random, P, L, c_uint64, I, F, F, P)
        _sig(lib.vk_pull, P, L, P, P)
        _sig(lib.vk_gemm, P, P, P, I, I, I, L, L, I, P)
        _sig(lib.vk_gemm_swiglu, P, P, P, I, I, I, L, L, P)
        _sig(lib.vk_gemm_swiglu_supported, I, I, I)
        _sig(lib.vk_gemm_split, P, P, P, I, I, I, L, L, I, P, L, P)
        lib.vk_gemm_split_floats.argtypes = [I, I, I, I]
        lib.vk_gemm_split_floats.restype = c_int64
        _sig(lib.vk_gemm_split_preferred, I, I, I, I)
        _sig(lib.vk_qkv_post, P, L, P, P, P, P, P, I, P, P, I, P, P, I, I, I, I, I, F, P)
        _sig(lib.vk_paged_attention, P, P, P, P, P, I, P, P, P, I, I, I, P, I, I, I, I, I, I, F, P)
        _sig(lib.vk_sample, P, P, P, P, P, I, I, L, P)
        lib.vk_sample_scratch_words.argtypes = [I]
        lib.vk_sample_scratch_words.restype = c_int
        lib.vk_attn_scratch_floats.argtypes = [I, I, I, I]
        lib.vk_attn_scratch_floats.restype = c_int64
        lib.vk_attn_segment_keys.restype = c_int
        assert lib.vk_attn_segment_keys() == SEGMENT_KEYS
        lib.vk_attn_item_rows.restype = c_int
        _sig(lib.vk_qkv_post8, P, L, P, P, P, P, P, P, I, P, P, I, P, I, P, P, I, I, I, I, I, I, I, I, c_double, P)
        _sig(lib.vk_paged_attention8, P, P, P, P, P, P, I, P, P, P, I, I, P, L, I, I, I, I, I, I, I, I, I, F, P)
        lib.vk_attn8_scratch_floats.argtypes = [I, I, I, I, I, I]
        lib.vk_attn8_scratch_floats.restype = c_int64
        _sig(lib.vk_verify, P, P, P, P, P, P, P, P, P, P, P, L, I, I, I, I, P)
        lib.vk_verify_scratch_bytes.argtypes = [I, I, I, I]
        lib.vk_verify_scratch_bytes.restype = c_int64
        assert lib.vk_attn_item_rows() == ATTN_ITEM_ROWS
        self.lib = lib

    # ------------------------------------------------------------ helpers
    def _call(self, fn, *args):
        if fn(*args) != 0:
            raise KernelError(self.lib.vk_last_error().decode())

    @staticmethod
    def _stream() -> int:
        return _raw_stream(torch.cuda.current_device()) if _raw_stream is not None else torch.cuda.current_stream().cuda_stream

    def _elem(self, t: torch.Tensor, what: str, *shape) -> int:
        self._check(t, what, self.dtype, shape)
        return t.data_ptr()

    @staticmethod
    def _check(t: torch.Tensor, what: str, dtype, shape=()) -> None:
        if not isinstance(t, torch.Tensor):
            raise KernelError(f"{what} is not a tensor")
        if not t.is_cuda:
            raise KernelError(f"{what} is not on the GPU")
        if t.dtype != dtype:
            raise KernelError(f"{what} has type {t.dtype}, expected {dtype}")
        if not t.is_contiguous():
            raise KernelError(f"{what} is not contiguous")
        if shape and t.shape != tuple(shape):
            raise KernelError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")

    def _i32(self, t: torch.Tensor, what: str, *shape) -> int:
        self._check(t, what, torch.int32, shape)
        return t.data_ptr()

    def _f32(self, t: torch.Tensor, what: str, *shape) -> int:
        self._check(t, what, torch.float32, shape)
        return t.data_ptr()

    def _weight(self, w: torch.Tensor, what: str, n: int) -> tuple[int, int]:
        """A norm weight may be stored as elements or as float."""
        if w.dtype == torch.float32 and self.dtype != torch.float32:
            self._check(w, what, torch.float32, (n,))
            return w.data_ptr(), 1
        self._check(w, what, self.dtype, (n,))
        return w.data_ptr(), 1 if self.dtype == torch.float32 else 0

    def empty(self, *shape) -> torch.Tensor:
        return torch.empty(shape, dtype=self.dtype, device="cuda")

    # ---------------------------------------------------------------- ops
    def embedding(self, table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """out[t] = table[ids[t]].  ids (int32, on the GPU) must lie in [0, V): the caller checks on the host."""
        V, H = table.shape
        T = ids.shape[0]
        out = self.empty(T, H) if out is None else out
        self._call(self.lib.vk_embedding, self._elem(out, "out", T, H), self._elem(table, "table", V, H),
                   self._i32(ids, "ids", T), T, H, V, self._stream())
        return out

    def rmsnorm(self, x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
        """Row-wise RMSNorm over the last axis of a contiguous tensor."""
        H = x.shape[-1]
        rows = x.numel() // H
        out = torch.empty_like(x) if out is None else out
        wp, wf = self._weight(w, "norm weight", H)
        self._call(self.lib.vk_rmsnorm, self._elem(out, "out", *x.shape), self._elem(x, "x"), wp, wf, rows, H, 1, H, H,
                   float(eps), self._stream())
        return out

    def add_rmsnorm(self, x: torch.Tensor, residual: torch.Tensor, w: torch.Tensor, eps: float,
                    out: torch.Tensor | None = None) -> torch.Tensor:
        """residual += x in place (fp32 sum, stored rounded); returns rmsnorm of the unrounded sum."""
        T, H = x.shape
        out = torch.empty_like(x) if out is None else out
        wp, wf = self._weight(w, "norm weight", H)
        self._call(self.lib.vk_add_rmsnorm, self._elem(out, "out", T, H), self._elem(residual, "residual", T, H),
                   self._elem(x, "x", T, H), wp, wf, T, H, float(eps), self._stream())
        return out

    def swiglu(self, gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        T, I2 = gate_up.shape
        if I2 % 2:
            raise KernelError(f"swiglu: width {I2} of the gate/up tensor is odd")
        I = I2 // 2
        out = self.empty(T, I) if out is None else out
        self._call(self.lib.vk_swiglu, self._elem(out, "out", T, I), self._elem(gate_up, "gate_up", T, I2), T, I,
                   self._stream())
        return out

    def gather_rows(self, x: torch.Tensor, rows: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """out[r] = x[rows[r]].  rows (int32, on the GPU) must lie in [0, T): the caller checks on the host."""
        T, H = x.shape
        R = rows.shape[0]
        out = self.empty(R, H) if out is None else out
        self._call(self.lib.vk_gather_rows, self._elem(out, "out", R, H), self._elem(x, "x", T, H),
                   self._i32(rows, "rows", R), R, H, self._stream())
        return out

    def to_f32(self, x: torch.Tensor) -> torch.Tensor:
        out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
        self._call(self.lib.vk_cast_to_f32, self._f32(out, "out"), self._elem(x, "x"), x.numel(), self._stream())
        return out

    def from_f32(self, x: torch.Tensor) -> torch.Tensor:
        out = torch.empty(x.shape, dtype=self.dtype, device=x.device)
        self._call(self.lib.vk_cast_from_f32, self._elem(out, "out"), self._f32(x, "x"), x.numel(), self._stream())
        return out

    def rope_tables(self, inv_freq: torch.Tensor, max_pos: int) -> tuple[torch.Tensor, torch.Tensor]:
        half = inv_freq.shape[0]
        cos, sin = self.empty(max_pos, half), self.empty(max_pos, half)
        self._call(self.lib.vk_rope_tables, cos.data_ptr(), sin.data_ptr(), self._f32(inv_freq, "inv_freq", half),
                   max_pos, half, self._stream())
        return cos, sin

    def pull(self, t: torch.Tensor, sink: torch.Tensor) -> None:
        """Reads ``t`` (contiguous) once and keeps nothing: the yardstick of what a kernel that must read it can
        reach.  ``sink``: an int32 tensor on the GPU that is practically never written."""
        if not t.is_contiguous() or not t.is_cuda:
            raise KernelError("pull: a contiguous tensor on the GPU is needed")
        self._call(self.lib.vk_pull, t.data_ptr(), t.numel() * t.element_size(), self._i32(sink, "sink"), self._stream())

    def fill_random(self, out: torch.Tensor, seed: int, kind: int, p0: float, p1: float) -> None:
        self._call(self.lib.vk_fill_random, self._elem(out, "out"), out.numel(), c_uint64(seed & (2**64 - 1)), kind,
                   float(p0), float(p1), self._stream())

    def gemm_workspace_floats(self, M: int, rows: int, K: int, swiglu: bool = False, force: bool = False) -> int:
        """float32 elements of workspace with which ``gemm`` / ``gemm_swiglu`` take the route through chunk
        sums for these sizes, or 0 where that route does not exist or is the slower one (``force``: where it
        does not exist).  A part adds this to what it asks of the step's workspace."""
        if not force and not self.lib.vk_gemm_split_preferred(M, rows, K, 1 if swiglu else 0):
            return 0
        return int(self.lib.vk_gemm_split_floats(M, rows, K, 1 if swiglu else 0))

    def _split(self, out, act, w, M, rows, K, lda, ldo, swiglu, workspace, force=False) -> bool:
        """Runs the product through chunk sums in ``workspace`` if that is the faster route and it fits."""
        if workspace is None:
            if force:
                raise KernelError("gemm: the route through chunk sums needs a workspace")
            return False
        need = self.gemm_workspace_floats(M, rows, K, swiglu, force)
        if need == 0 or workspace.numel() < need:
            if force:
                raise KernelError(f"gemm: no route through chunk sums for M={M} rows={rows} K={K}, or the workspace "
                                  f"of {workspace.numel()} floats is smaller than {need}")
            return False
        self._call(self.lib.vk_gemm_split, out.data_ptr(), act.data_ptr(), w.data_ptr(), M, rows, K, lda, ldo,
                   1 if swiglu else 0, self._f32(workspace, "workspace"), workspace.numel(), self._stream())
        return True

    def gemm(self, act: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None, kernel: int = 0,
             workspace: torch.Tensor | None = None) -> torch.Tensor:
        """out = act @ w.T with w in [out_features, in_features] layout.

        ``act`` may be a view of rows with a row stride (its last axis contiguous).  ``workspace``: float32
        scratch; with enough of it (``gemm_workspace_floats``) some sizes take a faster route to the same
        bits.  ``kernel`` 14 forces that route (tests)."""
        M, K = act.shape
        N, K2 = w.shape
        if K2 != K:
            raise KernelError(f"gemm: activation width {K} differs from the weight's input width {K2}")
        self._check(w, "weight", self.dtype, (N, K))
        if not act.is_cuda or act.dtype != self.dtype or act.stride(1) != 1:
            raise KernelError("gemm: activation must be a GPU tensor of the element type with a contiguous last axis")
        lda = act.stride(0) if M > 1 else max(K, act.stride(0))
        out = self.empty(M, N) if out is None else out
        self._elem(out, "out", M, N)
        if kernel in (0, 14) and self._split(out, act, w, M, N, K, lda, N, False, workspace, force=kernel == 14):
            return out
        self._call(self.lib.vk_gemm, out.data_ptr(), act.data_ptr(), w.data_ptr(), M, N, K, lda, N, kernel,
                   self._stream())
        return out

    def gemm_swiglu(self, act: torch.Tensor, w_gate_up: torch.Tensor, workspace: torch.Tensor | None = None,
                    split: bool = False) -> torch.Tensor:
        """silu(act @ w_gate.T) * (act @ w_up.T) with w_gate_up = [gate rows; up rows].

        One launch where the sizes allow it, else the projection and the activation one after the
        other; the result is the same bits either way.  ``split`` forces the route through chunk sums in
        ``workspace`` (tests)."""
        M, K = act.shape
        N2, K2 = w_gate_up.shape
        if K2 != K or N2 % 2:
            raise KernelError(f"gemm_swiglu: activation [{M}, {K}] does not fit a gate/up weight [{N2}, {K2}]")
        I = N2 // 2
        if not (act.is_contiguous() and self.lib.vk_gemm_swiglu_supported(M, I, K)):
            return self.swiglu(self.gemm(act, w_gate_up, workspace=workspace))
        self._elem(act, "activation", M, K)
        self._elem(w_gate_up, "weight", N2, K)
        out = self.empty(M, I)
        if self._split(out, act, w_gate_up, M, N2, K, K, I, True, workspace, force=split):
            return out
        self._call(self.lib.vk_gemm_swiglu, out.data_ptr(), act.data_ptr(), w_gate_up.data_ptr(), M, I, K, K, I,
                   self._stream())
        return out

    def qkv_post(self, qkv: torch.Tensor, *, nq: int, nkv: int, d: int, q_out: torch.Tensor | None,
                 k_cache: torch.Tensor | None, v_cache: torch.Tensor | None, page_size: int,
                 q_w: torch.Tensor | None, k_w: torch.Tensor | None, eps: float,
                 cos: torch.Tensor | None, sin: torch.Tensor | None, positions: torch.Tensor | None,
                 slots: torch.Tensor | None) -> torch.Tensor | None:
        """Head norm, rotation and cache store of a [T, (nq + 2 nkv) d] row tensor (see qkv_post.hip).

        Positions must be below the tables' row count and slots inside the caches: checked by the caller on the host."""
        T, W = qkv.shape
        if W != (nq + 2 * nkv) * d:
            raise KernelError(f"qkv_post: row width {W} is not (nq + 2 nkv) * d = {(nq + 2 * nkv) * d}")
        self._elem(qkv, "qkv", T, W)
        if nq:
            q_out = self.empty(T, nq, d) if q_out is None else q_out
            self._elem(q_out, "q_out", T, nq, d)
        wf = 0
        qwp = kwp = None
        if q_w is not None:
            qwp, wf = self._weight(q_w, "q norm weight", d)
        if k_w is not None:
            kwp, wf2 = self._weight(k_w, "k norm weight", d)
            if q_w is not None and wf2 != wf:
                raise KernelError("qkv_post: q and k norm weights must have the same type")
            wf = wf2
        rot_half = 0
        if cos is not None:
            max_pos, rot_half = cos.shape
            self._elem(cos, "cos", max_pos, rot_half)
            self._elem(sin, "sin", max_pos, rot_half)
            self._i32(positions, "positions", T)
        kcp = vcp = None
        if nkv:
            pages = k_cache.shape[0]
            kcp = self._elem(k_cache, "k cache", pages, nkv, page_size, d)
            vcp = self._elem(v_cache, "v cache", pages, nkv, d, page_size)
            self._i32(slots, "slots", T)
        self._call(self.lib.vk_qkv_post, qkv.data_ptr(), W, q_out.data_ptr() if nq else None, kcp, vcp, qwp, kwp, wf,
                   cos.data_ptr() if cos is not None else None, sin.data_ptr() if sin is not None else None, rot_half,
                   positions.data_ptr() if positions is not None else None,
                   slots.data_ptr() if slots is not None else None, T, nq, nkv, d, page_size, float(eps),
                   self._stream())
        return q_out

    def attn_scratch_floats(self, items: int, nq: int, d: int, nseg: int) -> int:
        """float32 elements of scratch that decode attention (mode 1) needs for ``items`` decoded tokens."""
        return int(self.lib.vk_attn_scratch_floats(items, nq, d, nseg))

    def paged_attention(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        block_table: torch.Tensor, cu_q: torch.Tensor, k_len: torch.Tensor, items: torch.Tensor,
                        *, mode: int, scale: float, window: int = 0, max_k_len: int,
                        nseg: int = 0, scratch: torch.Tensor | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the rows named by ``items`` over the paged cache (see attention.hip).

        items [n, 2] = (sequence, first row).  mode 0: an item is up to ATTN_ITEM_ROWS consecutive new
        rows of its sequence; modes 2, 6, 8 and 9: the same through a named kernel (same bits); mode 1: an item
        is a single decoded token; modes 3, 4, 5, 7: the same through a named kernel (same bits; see
        attention.hip).  ``max_k_len`` is the host's bound on k_len; the block table must cover it."""
        T, nq, d = q.shape
        pages, nkv, P, d2 = k_cache.shape
        S, W = block_table.shape
        self._elem(q, "q", T, nq, d)
        self._elem(k_cache, "k cache", pages, nkv, P, d)
        self._elem(v_cache, "v cache", pages, nkv, d, P)
        self._i32(block_table, "block table", S, W)
        self._i32(cu_q, "cu_q", S + 1)
        self._i32(k_len, "k_len", S)
        n_items = items.shape[0]
        self._i32(items, "items", n_items, 2)
        if W * P < max_k_len:
            raise KernelError(f"attention: block table of {W} pages of {P} does not cover {max_k_len} keys")
        out = torch.empty_like(q) if out is None else out
        self._elem(out, "out", T, nq, d)
        sp = None
        if mode in (1, 3, 4, 5, 7):
            need_seg = -(-max_k_len // SEGMENT_KEYS)
            if nseg < need_seg:
                raise KernelError(f"attention: {nseg} segments do not cover {max_k_len} keys")
            need = self.attn_scratch_floats(n_items, nq, d, nseg)
            if scratch is None or scratch.numel() < need:
                raise KernelError(f"attention: scratch of {need} floats needed")
            sp = self._f32(scratch, "scratch")
        self._call(self.lib.vk_paged_attention, out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                   block_table.data_ptr(), W, cu_q.data_ptr(), k_len.data_ptr(), items.data_ptr(), n_items, mode,
                   nseg, sp, T, nq, nkv, d, P, window, float(scale), self._stream())
        return out

    def sample(self, logits: torch.Tensor, temps: torch.Tensor | None = None, uniforms: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Token ids for each row: argmax, or temperature sampling where temps[r] > 0."""
        R, V = logits.shape
        self._elem(logits, "logits", R, V)
        out = torch.empty(R, dtype=torch.int32, device=logits.device) if out is None else out
        self._i32(out, "out", R)
        tp = up = None
        if temps is not None:
            tp, up = self._f32(temps, "temps", R), self._f32(uniforms, "uniforms", R)
        scratch = torch.empty(self.lib.vk_sample_scratch_words(R), dtype=torch.int32, device=logits.device)
        self._call(self.lib.vk_sample, out.data_ptr(), logits.data_ptr(), tp, up, scratch.data_ptr(), R, V, V,
                   self._stream())
        return out

    # ------------------------------------------------ caches of 8 bits, drafted tokens
    @staticmethod
    def _device() -> int:
        try:
            return torch.cuda.current_device()
        except (RuntimeError, AssertionError):          # no GPU: no tensor lies there
            return -2

    def _at(self, t: torch.Tensor, what: str, dtype, shape, here: int) -> int:
        """The address of a contiguous tensor of this type and shape on the current device (``here``: a launch goes there); anything else is refused."""
        if isinstance(t, torch.Tensor) and t.get_device() == here and t.dtype == dtype and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
        self._check(t, what, dtype)
        if t.shape != shape:
            raise KernelError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        raise KernelError(f"{what} lies on {t.device}, the current device is cuda:{here}")

    def empty_cache8(self, pages: int, nkv: int, page_size: int, d: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Keys [pages, nkv, page_size, d], values [pages, nkv, d, page_size] (both e4m3) and scales [pages, nkv, 2] of an empty 8-bit cache."""
        return (torch.zeros(pages, nkv, page_size, d, dtype=CACHE8_DTYPE, device="cuda"),
                torch.zeros(pages, nkv, d, page_size, dtype=CACHE8_DTYPE, device="cuda"),
                torch.zeros(pages, nkv, 2, dtype=torch.float32, device="cuda"))

    def _cache8(self, k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, nkv: int, d: int, here: int) -> tuple[int, int, int, int, int]:
        """Checks the three tensors; returns (pages, page size, their addresses)."""
        if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4:
            raise KernelError("k cache is no tensor [pages, kv heads, page size, head size]")
        pages, _, P, _ = k_cache.shape
        if P & (P - 1) or not CACHE8_PAGES[0] <= P <= CACHE8_PAGES[1]:
            raise KernelError(f"page size {P} of an 8-bit cache is no power of two from {CACHE8_PAGES[0]} to {CACHE8_PAGES[1]}")
        return (pages, P, self._at(k_cache, "k cache", CACHE8_DTYPE, (pages, nkv, P, d), here), self._at(v_cache, "v cache", CACHE8_DTYPE, (pages, nkv, d, P), here),
                self._at(scales, "scales", torch.float32, (pages, nkv, 2), here))

    def qkv_post8(self, qkv: torch.Tensor, *, nq: int, nkv: int, d: int, k_cache: torch.Tensor | None, v_cache: torch.Tensor | None,
                  scales: torch.Tensor | None, q_w: torch.Tensor | None, k_w: torch.Tensor | None, eps: float, cos: torch.Tensor | None,
                  sin: torch.Tensor | None, block_table: torch.Tensor, cu_q: torch.Tensor, k_len: torch.Tensor, max_k_len: int,
                  q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """``qkv_post`` for an 8-bit cache: head norm, rotation and append of a [T, (nq + 2 nkv) d] row tensor (see store8.hip).

        Rows of sequence s are cu_q[s] .. cu_q[s + 1] - 1 and stand at the places before k_len[s] (its keys with them) in the pages of
        block_table[s]; a page number outside the cache keeps nothing.  ``qkv`` may be a view of rows with a row stride that is a whole number of
        16-byte vectors.  A page's scales grow with its entries and start anew when a call writes its first place; a page that two sequences of a call write
        to is undefined.  ``max_k_len``: the host's bound on k_len, which tables and block tables cover; a sequence beyond it is left out.  Rows behind the
        last sequence's are left as they were."""
        here = self._device()
        if qkv.dim() != 2 or nq < 0 or nkv < 0 or qkv.shape[1] != (nq + 2 * nkv) * d:
            raise KernelError(f"qkv_post8: row tensor {tuple(qkv.shape)} is not [T, (nq + 2 nkv) * d = {(nq + 2 * nkv) * d}]")
        T, W = qkv.shape
        if qkv.get_device() != here or qkv.dtype != self.dtype or (W and qkv.stride(1) != 1):
            raise KernelError("qkv_post8: rows must be a tensor of the element type on the current GPU with a contiguous last axis")
        qp = kcp = vcp = scp = qwp = kwp = cp = sp = None
        pages = P = wf = half = 0
        if nq:
            q_out = torch.empty((T, nq, d), dtype=self.dtype, device=qkv.device) if q_out is None else q_out
            qp = self._at(q_out, "q_out", self.dtype, (T, nq, d), here)
        if q_w is not None and k_w is not None and q_w.dtype != k_w.dtype:
            raise KernelError("qkv_post8: q and k norm weights must have the same type")
        if q_w is not None:
            wf = int(q_w.dtype == torch.float32)
            qwp = self._at(q_w, "q norm weight", torch.float32 if wf else self.dtype, (d,), here)
        if k_w is not None:
            wf = int(k_w.dtype == torch.float32)
            kwp = self._at(k_w, "k norm weight", torch.float32 if wf else self.dtype, (d,), here)
        if cos is not None:
            if cos.dim() != 2 or cos.shape[0] < max_k_len:
                raise KernelError(f"qkv_post8: tables {tuple(cos.shape)} do not cover {max_k_len} places")
            half = cos.shape[1]
            cp, sp = self._at(cos, "cos", self.dtype, cos.shape, here), self._at(sin, "sin", self.dtype, cos.shape, here)
        if not 0 <= max_k_len < 2**31:
            raise KernelError(f"qkv_post8: up to {max_k_len} keys")
        S, width = block_table.shape
        tp = self._at(block_table, "block table", torch.int32, (S, width), here)
        cup, klp = self._at(cu_q, "cu_q", torch.int32, (S + 1,), here), self._at(k_len, "k_len", torch.int32, (S,), here)
        if nkv:
            pages, P, kcp, vcp, scp = self._cache8(k_cache, v_cache, scales, nkv, d, here)
        self._call(self.lib.vk_qkv_post8, qkv.data_ptr(), qkv.stride(0) if T > 1 else W, qp, kcp, vcp, scp, qwp, kwp, wf, cp, sp, half, tp, width, cup, klp, T, S,
                   nq, nkv, d, P, pages, max_k_len, eps, self._stream())
        return q_out if nq else None

    def attn8_scratch_floats(self, items: int, item_rows: int, nq: int, d: int, max_k_len: int, window: int = 0) -> int:
        """float32 elements of scratch that ``paged_attention8`` needs for ``items`` items of up to ``item_rows`` rows: items * item_rows * nq * (d + 2) for each segment of 512 keys, those of
        the bound or, with a window, those that window + item_rows - 1 neighbouring keys can touch.  (64 items of 5 rows, 64 heads of 128: 10.6 MB a segment, and 2.7 GB for a bound of 131,072
        keys without a window.)"""
        return int(self.lib.vk_attn8_scratch_floats(items, item_rows, nq, d, max_k_len, window))

    def paged_attention8(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor,
                         block_table: torch.Tensor, cu_q: torch.Tensor, k_len: torch.Tensor, items: torch.Tensor,
                         *, item_rows: int, scale: float, window: int = 0, max_k_len: int, scratch: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the rows named by ``items`` over an 8-bit cache (see attention8.hip).

        items [n, 2] = (sequence, first row): an item is up to ``item_rows`` consecutive rows of its sequence, at most ATTN_ITEM_ROWS.  Items of up
        to 16 rows have their keys split over workgroups, whose sums meet in ``scratch`` (``attn8_scratch_floats``; without it the call takes memory of its own);
        a scratch belongs to one call at a time, in recorded graphs too.  They are for decoded and drafted tokens and for a portion of few sequences (32 heads of 128,
        one sequence of 8,192 keys: 128 rows in 45 us, as one item in 180); larger items read the cache less often and are for prompts (1,024 rows of that sequence: 182 us
        against 247; 64 portions of 128 rows with 1,000 keys: 156 against 334).  A row's last bits depend on its item (``item_rows``, the item's other
        rows) and on nothing else in the call.  ``max_k_len`` is the host's bound on k_len; the block table must cover it, and keys beyond it may be left out.  Rows that no item
        names are left as they were.

        In bfloat16, weights are off by up to 2^-11 of themselves, or by 2^-32 of the row's largest where that is more; for heads of 80 to 128 and of 208 to 256 entries, entries of q below
        2^-14 of their head's largest are off by up to 2^-22 of it (heads of other sizes take q whole); and values of pages whose scale is 2^75 below that of another page that the same
        item sees may count as 0."""
        here = self._device()
        if q.dim() != 3 or k_cache.dim() != 4:
            raise KernelError(f"attention8: q {tuple(q.shape)} is not [T, heads, size], or the k cache {tuple(k_cache.shape)} not [pages, kv heads, page size, size]")
        if not 1 <= item_rows <= ATTN_ITEM_ROWS:
            raise KernelError(f"attention8: items of {item_rows} rows; from 1 to {ATTN_ITEM_ROWS}")
        if not 0 <= window < 2**31 or not 0 <= max_k_len < 2**31:
            raise KernelError(f"attention8: a window of {window}, up to {max_k_len} keys")
        T, nq, d = q.shape
        nkv = k_cache.shape[1]
        S, W = block_table.shape
        n_items = items.shape[0]
        qp = self._at(q, "q", self.dtype, (T, nq, d), here)
        pages, P, kcp, vcp, scp = self._cache8(k_cache, v_cache, scales, nkv, d, here)
        tp, cup = self._at(block_table, "block table", torch.int32, (S, W), here), self._at(cu_q, "cu_q", torch.int32, (S + 1,), here)
        klp, ip = self._at(k_len, "k_len", torch.int32, (S,), here), self._at(items, "items", torch.int32, (n_items, 2), here)
        out = torch.empty_like(q) if out is None else out
        op = self._at(out, "out", self.dtype, (T, nq, d), here)
        need, scratch_p = self.attn8_scratch_floats(n_items, item_rows, nq, d, max_k_len, window) if item_rows <= 16 else 0, None
        if need:
            scratch = torch.empty(need, dtype=torch.float32, device=q.device) if scratch is None else scratch
            scratch_p = self._at(scratch, "scratch", torch.float32, (scratch.numel(),), here)
        self._call(self.lib.vk_paged_attention8, op, qp, kcp, vcp, scp, tp, W, cup, klp, ip, n_items, item_rows, scratch_p, scratch.numel() if need else 0, T, S, nq, nkv, d,
                   P, pages, max_k_len, window, scale, self._stream())
        return out

    def verify(self, logits: torch.Tensor, draft_ids: torch.Tensor, cu: torch.Tensor, *, draft_logits: torch.Tensor | None = None,
               temps: torch.Tensor | None = None, accept_uniforms: torch.Tensor | None = None,
               draw_uniforms: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Which drafted tokens stand against the target's logits, and the token behind them (see verify.hip).

        logits [R, V]: rows cu[s] .. cu[s + 1] - 1 (cu[0] = 0) are sequence s's, one more than its drafted tokens; draft_ids [D] are those of all sequences one after
        the other.  ``draft_logits`` [D, V]: the draft model's, without them a draft is certain.  ``temps`` [S] for both models (without them, and at 0, the
        maximum alone), with random numbers in [0, 1): ``accept_uniforms`` [D] and ``draw_uniforms`` [S].

        Returns (tokens [R], counts [S], accept [D]): sequence s's rows of ``tokens`` begin with counts[s] tokens (the standing ones and the drawn one) and go on
        with -1; ``accept`` is min(1, p / q) of every drafted token.  What lies behind the last sequence is not written."""
        here = self._device()
        if logits.dim() != 2 or draft_ids.dim() != 1 or cu.dim() != 1 or cu.shape[0] < 1:
            raise KernelError(f"verify: logits {tuple(logits.shape)}, draft ids {tuple(draft_ids.shape)} and cu {tuple(cu.shape)} are not [R, V], [D], [S + 1]")
        R, V = logits.shape
        D, S = draft_ids.shape[0], cu.shape[0] - 1
        lp, ip, cup = self._at(logits, "logits", self.dtype, (R, V), here), self._at(draft_ids, "draft ids", torch.int32, (D,), here), self._at(cu, "cu", torch.int32, (S + 1,), here)
        dp = self._at(draft_logits, "draft logits", self.dtype, (D, V), here) if draft_logits is not None else None
        tp = ap = up = None
        if temps is not None:
            if accept_uniforms is None or draw_uniforms is None:
                raise KernelError("verify: temperatures need random numbers")
            tp, ap = self._at(temps, "temps", torch.float32, (S,), here), self._at(accept_uniforms, "accept uniforms", torch.float32, (D,), here)
            up = self._at(draw_uniforms, "draw uniforms", torch.float32, (S,), here)
        dev = logits.device
        tokens, counts = torch.empty(R, dtype=torch.int32, device=dev), torch.empty(S, dtype=torch.int32, device=dev)
        accept = torch.empty(D, dtype=torch.float32, device=dev)
        need = self.lib.vk_verify_scratch_bytes(R, D, S, V)
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        self._call(self.lib.vk_verify, tokens.data_ptr(), counts.data_ptr(), accept.data_ptr(), lp, ip, cup, dp, tp, ap, up, scratch.data_ptr(), need, R, D, S, V,
                   self._stream())
        return tokens, counts, accept


_CACHE: dict[str, Kernels] = {}


def kernels_for(dtype) -> Kernels:
    name = dtype_name(dtype)
    if name not in _CACHE:
        _CACHE[name] = Kernels(name)
    return _CACHE[name]
