"""Paged 4-bit KV cache over torch tensors: planning a step, storing and loading rows, attention (include/faie2fn.h,
fn_kv4_*). The reference keeps one dense fp32 cache per layer and steps all tokens at one position
(engine/faie2fn.cu:1452-1690); this is for batches of requests of different lengths whose pages come and go.

    fn = FN()
    planner = KV4Planner(fn, page_size=64)                    # one per server: pages serve every layer alike
    cache = KV4Cache(fn, nkv=2, hd=256, page_size=64, pages=4096)   # one per attention layer
    step = planner.plan(ctx, add, table, free, free_count, max_tokens=32)
    cache.store(k, v, step.slots)                             # [rows][nkv][hd], fp32 or bf16, any token / head stride
    out = cache.attn(q, step.cu, step.kv_len, table, max_new=1, gate=g)
    ctx.copy_(step.ctx)                                       # the next step's inputs: a served request's new length, 0 of a
    free_count.copy_(step.free_count)                         # finished one, the old one of a refused one (its pages stay its own)

Everything runs on the current stream and returns at once; arguments that the kernels cannot check are the device-side
lengths and page ids, which they clamp to the tensors' bounds.
"""

from __future__ import annotations

import ctypes as C
import math

import torch

from fn import FnKv4

F32, BF16 = 0, 30  # ggml type ids of rows
GROUP = 64         # dims that share a scale
_TYPE = {torch.float32: F32, torch.bfloat16: BF16}


def record_bytes(hd: int, page_size: int) -> int:
    """Bytes of one kv head's page: codes and scales of its keys and values."""
    return 2 * page_size * (hd // 2 + hd // GROUP * 2)


class Fixed:
    """Attributes named in FIXED are set once: pointers that calls pass were taken from them."""
    FIXED: frozenset = frozenset()

    def __setattr__(self, name, value):
        if name in self.FIXED and name in self.__dict__:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: make another {type(self).__name__}")
        super().__setattr__(name, value)


def _stream(dev) -> int:
    index = dev.index
    if torch.cuda.current_device() != index:  # kernels launch on the current device
        raise ValueError(f"the tensors are on {dev}: make it the current device")
    return torch._C._cuda_getCurrentRawStream(index)  # torch.cuda.current_stream().cuda_stream without its 2 us


def _ints(name, t, shape, dev):
    """dev: the index of the CUDA device that the call's tensors are on."""
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.get_device() != dev or dev < 0:
        raise ValueError(f"{name}: a contiguous int32 tensor {tuple(shape)} on cuda:{max(dev, 0)} is wanted, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


class KV4Plan(Fixed):
    """A planned step (device tensors): cu [n + 1], kv_len [n] (what attention reads: 0 for a refused request), ctx [n] (the lengths that
    requests go on with: a refused one's is unchanged), slots / positions / requests [max_tokens], free_count and status (refused
    requests), one value each."""
    FIXED = frozenset(("cu", "kv_len", "ctx", "slots", "positions", "requests", "free_count", "status", "ptrs"))

    def __init__(self, n, max_tokens, dev):
        ints = torch.empty(3 * n + 3 + 2 * max_tokens, dtype=torch.int32, device=dev)
        self.cu, self.kv_len, self.ctx, self.free_count, self.status, self.positions, self.requests = ints.split(
            [n + 1, n, n, 1, 1, max_tokens, max_tokens])
        self.slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
        self.ptrs = [t.data_ptr() for t in (self.cu, self.kv_len, self.slots, self.positions, self.requests, self.status, self.ctx)]


class KV4Planner:
    """Plans steps over pages of page_size tokens. Its outputs are the planner's buffers for that (requests, max_tokens):
    the next plan of the same sizes overwrites them (so a captured step always finds them in place); pass `out` (a
    KV4Plan) to own them."""

    def __init__(self, fn, page_size: int):
        self.fn, self.page_size, self.kept = fn, page_size, {}

    def plan(self, ctx, add, table, free, free_count, max_tokens: int, out: KV4Plan | None = None) -> KV4Plan:
        """ctx, add int32 [n]; table int32 [n][max_pages] and free int32 [pages] are updated in place; free_count int32
        [1] is read, the pages left are the plan's free_count."""
        n = ctx.numel()
        if table.dim() != 2:
            raise ValueError("table: [requests][max_pages] is wanted")
        dev = ctx.get_device()
        _ints("ctx", ctx, (n,), dev)
        _ints("add", add, (n,), dev)
        _ints("table", table, (n, table.shape[1]), dev)
        _ints("free", free, (free.numel(),), dev)
        _ints("free_count", free_count, (1,), dev)
        if out is None:
            key = (n, max_tokens, ctx.device)
            out = self.kept.get(key)
            if out is None:
                out = self.kept[key] = KV4Plan(n, max_tokens, ctx.device)
        elif out.kv_len.numel() != n or out.slots.numel() != max_tokens or out.slots.get_device() != dev:
            raise ValueError("out: a plan of other sizes, or on another device")
        cu, kv_len, slots, positions, requests, status, following = out.ptrs
        self.fn.kv4_plan(n, ctx.data_ptr(), add.data_ptr(), table.data_ptr(), table.shape[1], self.page_size,
                         free.data_ptr(), free.numel(), free_count.data_ptr(), out.free_count.data_ptr(), max_tokens, cu,
                         kv_len, slots, positions, requests, status, _stream(ctx.device), following)
        return out


class KV4Workspace(Fixed):
    """Scratch of the attention (split requests' partial results). Calls that may run at the same time, as on two
    streams, need one each."""
    FIXED = frozenset(("tensor", "ptr", "bytes"))

    def __init__(self, fn, device="cuda"):
        self.bytes = fn.kv4_attn_workspace()
        self.tensor = torch.empty(self.bytes, dtype=torch.uint8, device=device)
        self.ptr = self.tensor.data_ptr()


class KV4Cache(Fixed):
    """Pages of one attention layer. pages: their number (a zeroed uint8 tensor [pages][nkv][record_bytes] is made), or
    that tensor."""
    FIXED = frozenset(("pages", "nkv", "hd", "page_size"))

    def __init__(self, fn, nkv: int, hd: int, page_size: int, pages, workspace: KV4Workspace | None = None):
        if isinstance(pages, int):
            pages = torch.zeros(pages, nkv, record_bytes(hd, page_size), dtype=torch.uint8, device="cuda")
        if pages.dtype != torch.uint8 or not pages.is_contiguous() or not pages.is_cuda or \
                pages.shape[1:] != (nkv, record_bytes(hd, page_size)):
            raise ValueError("pages: a contiguous uint8 CUDA tensor [pages][nkv][record_bytes(hd, page_size)] is wanted")
        self.fn, self.nkv, self.hd, self.page_size, self.pages, self.dev = fn, nkv, hd, page_size, pages, pages.device
        self.ws = workspace or KV4Workspace(fn, self.dev)
        if self.ws.tensor.device != self.dev:
            raise ValueError(f"workspace: one on {self.dev} is wanted")
        self.index = pages.get_device()
        self.c = C.byref(FnKv4(pages.data_ptr(), pages.shape[0], page_size, nkv, hd))
        self.scale = 1.0 / math.sqrt(hd)
        self._store, self._load, self._attn = fn.kv4_store, fn.kv4_load, fn.kv4_attn

    def _rows(self, name, x, heads):
        s = x.shape
        if len(s) != 3 or s[1] != heads or s[2] != self.hd or x.stride(2) != 1 or x.dtype not in _TYPE or x.device != self.dev:
            raise ValueError(f"{name}: fp32 or bf16 [rows][{heads}][{self.hd}] on {self.dev} with adjacent dims is wanted, got "
                             f"{x.dtype} {tuple(s)}")

    def store(self, k, v, slots):
        """Quantise rows k, v [rows][nkv][hd] (any token and head stride) into their slots (int64 [rows]; < 0: skipped)."""
        self._rows("k", k, self.nkv)
        self._rows("v", v, self.nkv)
        nt = k.shape[0]
        if v.shape[0] != nt or v.dtype != k.dtype:
            raise ValueError("k, v: the same rows and type are wanted")
        self._slots(slots, nt)
        kt, kh, _ = k.stride()
        vt, vh, _ = v.stride()
        self._store(self.c, _TYPE[k.dtype], k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, slots.data_ptr(), nt, _stream(self.dev))

    def load(self, slots, dtype=torch.float32):
        """(k, v) [rows][nkv][hd], the values that slots stand for (zeros for slots < 0)."""
        if dtype not in _TYPE:
            raise ValueError("dtype: fp32 or bf16 is wanted")
        nt = slots.numel()
        self._slots(slots, nt)
        k = torch.empty(nt, self.nkv, self.hd, dtype=dtype, device=self.dev)
        v = torch.empty_like(k)
        self._load(self.c, _TYPE[dtype], slots.data_ptr(), nt, k.data_ptr(), v.data_ptr(), _stream(self.dev))
        return k, v

    def _slots(self, slots, nt):
        if slots.dtype != torch.int64 or slots.shape != (nt,) or not slots.is_contiguous() or slots.device != self.dev:
            raise ValueError(f"slots: a contiguous int64 tensor [{nt}] on {self.dev} is wanted")

    def attn(self, q, cu, kv_len, table, max_new: int, gate=None, scale: float | None = None, out=None):
        """Attention of the rows q [rows][nh][hd] of n requests over their pages: cu int32 [n + 1], kv_len int32 [n], table
        int32 [n][max_pages]; max_new: the most rows of a request (or a bound). gate: like q, out *= sigmoid(gate).
        scale: 1 / sqrt(hd) unless given. Returns out [rows][nh][hd] of q's type."""
        rows, nh = q.shape[0], q.shape[1]
        self._rows("q", q, nh)
        n = kv_len.numel()
        _ints("kv_len", kv_len, (n,), self.index)
        _ints("cu", cu, (n + 1,), self.index)
        _ints("table", table, (n, table.shape[-1]), self.index)
        if out is None:
            out = torch.empty(rows, nh, self.hd, dtype=q.dtype, device=self.dev)
        else:
            self._rows("out", out, nh)
            if out.shape != q.shape or out.dtype != q.dtype or out.stride(1) != self.hd:
                raise ValueError("out: q's shape and type with adjacent heads is wanted")
        g, gt, gh = None, 0, 0
        if gate is not None:
            self._rows("gate", gate, nh)
            if gate.shape != q.shape or gate.dtype != q.dtype:
                raise ValueError("gate: q's shape and type is wanted")
            g, gt, gh = gate.data_ptr(), gate.stride(0), gate.stride(1)
        self._attn(self.c, _TYPE[q.dtype], n, rows, nh, q.data_ptr(), q.stride(0), q.stride(1), g, gt, gh,
                         out.data_ptr(), out.stride(0), cu.data_ptr(), kv_len.data_ptr(), table.data_ptr(),
                         table.shape[1], max_new, self.scale if scale is None else scale, self.ws.ptr, self.ws.bytes,
                         _stream(self.dev))
        return out
