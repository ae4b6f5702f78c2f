"""A paged key/value cache held in 4 bits, on torch tensors: the sl_kv4_* operators of include/seedless_hip.h, which says
what each computes, refuses and leaves alone.

    pool = kv4.new_pool(n_pages, page_size, n_kv, head_dim)
    step = kv4.plan(ctx_len, new_len, table, held, free, free_count, page_size, max_tokens)     # once per step
    q = kv4.append(pool, q, k, v, step.slot, step.pos, cos, sin, q_weight, k_weight)            # per attention layer
    out = kv4.attention(pool, q, step.table, step.q_start, step.kv_len, max_rows=..., max_keys=...)

torch only owns the memory.  Calls enqueue on torch's current stream of the tensors' device and return without waiting;
they can be captured into a graph.  A call that the library refuses raises SeedlessError, a tensor of the wrong kind
ValueError; nothing is copied or converted on the way.  The operators have no gradients: a tensor that asks for one is refused
outside torch.no_grad().
"""
import ctypes as C
from typing import NamedTuple

import torch

from . import abi, lib as _lib

_DTYPES = {torch.float16: abi.SL_F16, torch.bfloat16: abi.SL_BF16}


class Pool(NamedTuple):
    """Pages of one layer's cache: `pages` uint8 [n_pages, page_size * n_kv * 9/8 * head_dim]."""
    pages: torch.Tensor
    page_size: int
    n_kv: int
    head_dim: int


class Plan(NamedTuple):
    table: torch.Tensor        # [n_req, width] page ids, -1 behind the used ones
    held: torch.Tensor         # [n_req] pages that each request holds
    free: torch.Tensor         # [n_free] free pages, -1 behind them
    free_count: torch.Tensor   # [1]
    q_start: torch.Tensor      # [n_req + 1] first row of each request
    kv_len: torch.Tensor       # [n_req] tokens in the cache once the new ones are stored; 0: not served
    slot: torch.Tensor         # [max_tokens] where each row's token goes, or -1
    pos: torch.Tensor          # [max_tokens] its position
    unserved: torch.Tensor     # [1] requests that did not get their pages


_page_bytes = {}


def page_bytes(page_size, n_kv, head_dim):
    layout = (page_size, n_kv, head_dim)
    n = _page_bytes.get(layout)
    if n is None:
        n = _lib.get().dll.sl_kv4_page_bytes(*layout)
        if not n:
            raise ValueError(f"no such layout: pages of {page_size} tokens, {n_kv} heads of {head_dim} dims")
        _page_bytes[layout] = n
    return n


def new_pool(n_pages, page_size, n_kv, head_dim, device="cuda"):
    return Pool(torch.empty(n_pages, page_bytes(page_size, n_kv, head_dim), dtype=torch.uint8, device=device), page_size, n_kv, head_dim)


def rope_tables(max_pos, rot_dim, theta=1e7, device="cuda"):
    """cos and sin [max_pos, rot_dim/2] of pos * theta^(-2i/rot_dim); angles in double precision, so that far positions
    keep theirs."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * torch.exp(i * (-2.0 / rot_dim) * torch.log(torch.tensor(theta, dtype=torch.float64)))
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _flat(t, shape, dtype, device, what):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: a tensor is wanted")
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: {dtype} {list(shape)} side by side on {device} is wanted, got {t.dtype} {list(t.shape)} on {t.device}")
    _no_grad(t, what)
    return t.data_ptr()


def _tensors(**named):
    for what, t in named.items():
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what}: a tensor is wanted")


def _no_grad(t, what):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and the operators on the 4-bit cache have none: detach it, or call under torch.no_grad()")


def _rows(t, shape, dtype, device, what):
    """Address and strides of [tokens, heads, dims] with the dims side by side."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: a tensor is wanted")
    token, head, dim = t.stride() if t.dim() == 3 else (0, 0, 0)
    if t.dtype is not dtype or t.shape != shape or t.device != device or dim != 1:
        raise ValueError(f"{what}: {dtype} {list(shape)} with dims side by side on {device} is wanted, got {t.dtype} {list(t.shape)} "
                         f"with strides {t.stride()} on {t.device}")
    _no_grad(t, what)
    return t.data_ptr(), token if shape[0] > 1 else 0, head if shape[1] > 1 else 0


def _pool(pool):
    p, page_size, n_kv, head_dim = pool
    _tensors(pages=p)
    n = page_bytes(page_size, n_kv, head_dim)
    if p.dtype is not torch.uint8 or not p.is_cuda or p.dim() != 2 or p.shape[1] != n or not p.is_contiguous():
        raise ValueError(f"pages: uint8 [n_pages, {n}] side by side on a GPU is wanted, got {p.dtype} {list(p.shape)} on {p.device}")
    return abi.Kv4Pool(p.data_ptr(), p.shape[0], page_size, n_kv, head_dim)


# The current stream's handle without a Stream object around it (2 us of a call's 15), where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_functions = {}


def _call(name, device, *args):
    """The library's call on torch's current stream of `device`, with that device current."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.get().dll, name)
    index = device.index
    if torch.cuda.current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.Library.check(status, name)


def plan(ctx_len, new_len, table, held, free, free_count, page_size, max_tokens, out=None):
    """sl_kv4_plan: page tables, slots and row offsets of one step from the requests' lengths (int32 tensors).  `out`: a
    Plan whose tensors are written, none of which may be an input; without it they come as parts of one new tensor."""
    _tensors(ctx_len=ctx_len, table=table, free=free)
    dev, i32 = ctx_len.device, torch.int32
    if not ctx_len.is_cuda or ctx_len.dim() != 1 or table.dim() != 2 or free.dim() != 1 or max_tokens < 0:
        raise ValueError("lengths [n_req], table [n_req, width] and free [n_free] on a GPU are wanted")
    n, width, n_free = ctx_len.shape[0], table.shape[1], free.shape[0]
    lengths = (n,)
    ins = (_flat(ctx_len, lengths, i32, dev, "ctx_len"), _flat(new_len, lengths, i32, dev, "new_len"), _flat(table, (n, width), i32, dev, "table"),
           _flat(held, lengths, i32, dev, "held"), _flat(free, (n_free,), i32, dev, "free"), _flat(free_count, (1,), i32, dev, "free_count"))
    sizes = (n * width, n, n_free, 1, n + 1, n, max_tokens, max_tokens, 1)
    if out is None:
        whole = torch.empty(sum(sizes), dtype=i32, device=dev)
        parts = whole.split_with_sizes(sizes)
        out = Plan(parts[0].view(n, width), *parts[1:])
        at, outs = whole.data_ptr(), []
        for size in sizes:
            outs.append(at)
            at += 4 * size
    else:
        outs = [_flat(t, (n, width) if i == 0 else (sizes[i],), i32, dev, "out." + Plan._fields[i]) for i, t in enumerate(out)]
    _call("sl_kv4_plan", dev, abi.Kv4PlanArgs(n, width, n_free, page_size, max_tokens, *ins, *outs))
    return out


def append(pool, q, k, v, slot, pos, cos, sin, q_weight, k_weight, eps=1e-6, out=None):
    """sl_kv4_append: queries normed and rotated are returned, keys normed and rotated and values go into the pool.  q None:
    keys and values only; cos and sin None: no rotation; a weight None: no norm."""
    p, dev = _pool(pool), pool.pages.device
    _tensors(k=k)
    if k.dtype not in _DTYPES or k.dim() != 3:
        raise ValueError(f"keys [tokens, heads, dims] in float16 or bfloat16 are wanted, got {k.dtype} {list(k.shape)}")
    dt, n, dim = k.dtype, k.shape[0], pool.head_dim
    kv, i32 = (n, pool.n_kv, dim), torch.int32
    k_at, v_at, q_at, out_at = _rows(k, kv, dt, dev, "k"), _rows(v, kv, dt, dev, "v"), (None, 0, 0), (None, 0, 0)
    heads = max_pos = rot = 0
    cos_at = sin_at = pos_at = qw_at = kw_at = None
    if q is not None:
        _tensors(q=q)
        heads = q.shape[1] if q.dim() == 3 else 0
        shape = (n, heads, dim)
        if out is None:
            out = torch.empty(shape, dtype=dt, device=dev)
        q_at, out_at = _rows(q, shape, dt, dev, "q"), _rows(out, shape, dt, dev, "out")
        if q_weight is not None:
            qw_at = _flat(q_weight, (dim,), dt, dev, "q_weight")
    if k_weight is not None:
        kw_at = _flat(k_weight, (dim,), dt, dev, "k_weight")
    if (cos is None) != (sin is None) or (cos is not None and not (isinstance(cos, torch.Tensor) and cos.dim() == 2)):
        raise ValueError("cos and sin [positions, rotated dims / 2] are wanted, or neither")
    if cos is not None:
        max_pos, rot = cos.shape[0], 2 * cos.shape[1]
        cos_at, sin_at, pos_at = _flat(cos, cos.shape, torch.float32, dev, "cos"), _flat(sin, cos.shape, torch.float32, dev, "sin"), _flat(pos, (n,), i32, dev, "pos")
    _call("sl_kv4_append", dev, p, abi.Kv4AppendArgs(n, heads, rot, max_pos, _DTYPES[dt], 0, eps, q_at[0], k_at[0], v_at[0], qw_at, kw_at, cos_at, sin_at,
                                                     _flat(slot, (n,), i32, dev, "slot"), pos_at, out_at[0], *q_at[1:], *k_at[1:], *v_at[1:], *out_at[1:]))
    return out


def _workspace(device, p, a):
    """(The library cuts a call by the current device's compute units.)"""
    size = _lib.get().dll.sl_kv4_attention_workspace
    if torch.cuda.current_device() == device.index:
        return size(p, a)
    with torch.cuda.device(device):
        return size(p, a)


def attention(pool, q, table, q_start, kv_len, max_rows, max_keys, scale=None, gate=None, out=None, workspace=None):
    """sl_kv4_attention: q [tokens, heads, dims] against the pages of each request; `workspace` (uint8, of at least
    attention_workspace() bytes) is taken from torch if it is not given.  Rows that no request has are not written: in
    a new `out` they hold whatever the memory held."""
    p, dev = _pool(pool), pool.pages.device
    _tensors(q=q, table=table)
    if q.dtype not in _DTYPES or q.dim() != 3 or table.dim() != 2:
        raise ValueError(f"queries [tokens, heads, dims] in float16 or bfloat16 and a table [n_req, width] are wanted, got {q.dtype} {list(q.shape)}, {list(table.shape)}")
    n, heads, n_req, dim = q.shape[0], q.shape[1], table.shape[0], pool.head_dim
    shape, dt = (n, heads, dim), q.dtype
    if out is None:
        out = torch.empty(shape, dtype=dt, device=dev)
    i32 = torch.int32
    q_at, out_at, gate_at = _rows(q, shape, dt, dev, "q"), _rows(out, shape, dt, dev, "out"), (None, 0, 0)
    if gate is not None:
        gate_at = _rows(gate, shape, dt, dev, "gate")
    max_rows, max_keys = min(max_rows, n), min(max_keys, 0x7fffffff)      # (the struct's are 32 bits)
    a = abi.Kv4AttnArgs(n_req, n, heads, _DTYPES[dt], table.shape[1], max_rows, max_keys, dim ** -0.5 if scale is None else scale, q_at[0], gate_at[0], out_at[0],
                        *q_at[1:], *gate_at[1:], *out_at[1:], _flat(table, table.shape, i32, dev, "table"), _flat(q_start, (n_req + 1,), i32, dev, "q_start"),
                        _flat(kv_len, (n_req,), i32, dev, "kv_len"))
    need = _workspace(dev, p, a)
    if need > 0:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif not isinstance(workspace, torch.Tensor) or workspace.dtype is not torch.uint8 or workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("workspace: uint8 side by side on the pool's device is wanted")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    _call("sl_kv4_attention", dev, p, a)
    return out


def attention_workspace(pool, n_tokens, n_heads, n_req, table_width, max_rows, max_keys):
    """Bytes of workspace that attention() takes for such a call (0: a call that has nothing to do, or is refused)."""
    a = abi.Kv4AttnArgs(n_req=n_req, n_tokens=n_tokens, n_heads=n_heads, table_width=table_width, max_rows=min(max_rows, n_tokens), max_keys=min(max_keys, 0x7fffffff))
    return _workspace(pool.pages.device, _pool(pool), a)


def read(pool, slots, dtype=torch.float32):
    """sl_kv4_read: keys and values [n, n_kv, head_dim] (float32 or float16) of the given slots."""
    p, dev = _pool(pool), pool.pages.device
    _tensors(slots=slots)
    if slots.dim() != 1 or dtype not in (torch.float32, torch.float16):
        raise ValueError("slots [n] and float32 or float16 values are wanted")
    n = slots.shape[0]
    k, v = (torch.empty(n, pool.n_kv, pool.head_dim, dtype=dtype, device=dev) for _ in range(2))
    _call("sl_kv4_read", dev, p, _flat(slots, (n,), torch.int32, dev, "slots"), n, abi.SL_F32 if dtype is torch.float32 else abi.SL_F16, k.data_ptr(), v.data_ptr())
    return k, v
