"""Torch-tensor wrappers over the C ABI, one per kernel entry point.

Each wrapper checks shapes, dtypes and devices on the host, then launches on
the current CUDA stream. Workspaces are plain zero-filled uint8 tensors the
caller keeps (the kernels leave them zeroed).
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib as L


def _ws(nbytes: int, device) -> torch.Tensor:
    return torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def status_tensor(device) -> torch.Tensor:
    return torch.zeros(1, dtype=torch.int32, device=device)


def check_status(status: torch.Tensor) -> None:
    """Raise if a kernel recorded a device-side error (syncs on `status`)."""
    code = int(status.item())
    if code != 0:
        status.zero_()
        raise L.KveError(code, "device-side check failed (see the op that wrote dev_status)")


class Workspace:
    """A grow-only zero-filled device scratch buffer."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.buf = _ws(256, self.device)

    def get(self, nbytes: int) -> torch.Tensor:
        if nbytes > self.buf.numel():
            self.buf = _ws(int(nbytes * 1.25) + 4096, self.device)
        return self.buf


def greedy_accept(logits: torch.Tensor, drafts: torch.Tensor, workspace: Workspace | None = None,
                  status: torch.Tensor | None = None, out=None):
    """logits [B, k+1, V] (fp32/bf16), drafts [B, k] (any int strides) ->
    (preds [B, k+1], n_accepted [B], emitted [B, k+1]) int32. `out` may give
    the three contiguous int32 result tensors (they may be views of one buffer,
    so that a single copy reads n_accepted and emitted back)."""
    lib = L.load()
    L.require_cuda(logits, drafts)
    B, kp1, V = logits.shape
    k = kp1 - 1
    if drafts.dtype != torch.int32 or tuple(drafts.shape) != (B, k):
        raise ValueError("drafts must be int32 [B, k]")
    if logits.stride(2) != 1 or logits.stride(0) != kp1 * logits.stride(1):
        raise ValueError("logits rows must be evenly strided with unit column stride")
    dev = logits.device
    if out is None:
        preds = torch.empty(B, kp1, dtype=torch.int32, device=dev)
        n_acc = torch.empty(B, dtype=torch.int32, device=dev)
        emitted = torch.empty(B, kp1, dtype=torch.int32, device=dev)
    else:
        preds, n_acc, emitted = out
        for t, shape in ((preds, (B, kp1)), (n_acc, (B,)), (emitted, (B, kp1))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != dev:
                raise ValueError("greedy_accept out tensors must be contiguous int32 on the logits' device")
    ws = (workspace or Workspace(dev)).get(lib.kve_greedy_accept_workspace_bytes(B))
    L.check(lib.kve_greedy_accept(
        logits.data_ptr(), L.dtype_code(logits.dtype), logits.stride(1), drafts.data_ptr(),
        drafts.stride(0), drafts.stride(1), B, k, V, preds.data_ptr(), n_acc.data_ptr(),
        emitted.data_ptr(), ws.data_ptr(), ws.numel(), L.ptr(status), L.stream_handle(dev)))
    return preds, n_acc, emitted


def argmax_rows(x: torch.Tensor, out: torch.Tensor | None = None, scatter_index: torch.Tensor | None = None,
                scatter_out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """int32 argmax of every row (first index on ties, NaN largest). With
    `scatter_index` / `scatter_out` (contiguous int32), row i's result is also
    written to scatter_out[scatter_index[i]]."""
    lib = L.load()
    L.require_cuda(x)
    rows, cols = x.shape
    if x.stride(1) != 1:
        raise ValueError("argmax_rows needs unit column stride")
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=x.device)
    if scatter_out is None:
        L.check(lib.kve_argmax_rows(x.data_ptr(), L.dtype_code(x.dtype), rows, cols, x.stride(0),
                                    out.data_ptr(), L.stream_handle(x.device)))
        return out
    for t in (scatter_index, scatter_out):
        if t.dtype != torch.int32 or not t.is_contiguous() or not t.is_cuda:
            raise ValueError("argmax_rows: scatter_index and scatter_out must be contiguous int32 CUDA tensors")
    if scatter_index.numel() != rows:
        raise ValueError("argmax_rows: one scatter index per row")
    L.check(lib.kve_argmax_rows_scatter(x.data_ptr(), L.dtype_code(x.dtype), rows, cols, x.stride(0),
                                        out.data_ptr(), scatter_index.data_ptr(), scatter_out.data_ptr(),
                                        scatter_out.numel(), L.ptr(status), L.stream_handle(x.device)))
    return out


def kv_append(k_new, v_new, slot_ids, pool_k_layer, pool_v_layer, status=None) -> None:
    """pool[slot] = new rows; pool_*_layer: [num_blocks, bs, nkv, hd] (one layer)."""
    lib = L.load()
    L.require_cuda(k_new, v_new, slot_ids, pool_k_layer, pool_v_layer)
    n, nkv, hd = k_new.shape
    num_slots = pool_k_layer.shape[0] * pool_k_layer.shape[1]
    for t in (k_new, v_new, pool_k_layer, pool_v_layer):
        if not t.is_contiguous() or t.dtype != k_new.dtype:
            raise ValueError("kv_append operands must be contiguous and share a dtype")
    if slot_ids.dtype != torch.int64:
        raise ValueError("slot_ids must be int64 (as index_copy_ takes)")
    L.check(lib.kve_kv_append(k_new.data_ptr(), v_new.data_ptr(), L.dtype_code(k_new.dtype),
                              slot_ids.data_ptr(), n, nkv, hd, pool_k_layer.data_ptr(),
                              pool_v_layer.data_ptr(), num_slots, L.ptr(status),
                              L.stream_handle(k_new.device)))


def qkv_rope_append(qkv, positions, slots, rope_cos, rope_sin, q_out, pool_k_layer, pool_v_layer,
                    num_heads, num_kv_heads, head_dim, status=None) -> None:
    lib = L.load()
    n = qkv.shape[0]
    num_slots = pool_k_layer.shape[0] * pool_k_layer.shape[1]
    L.check(lib.kve_qkv_rope_append(qkv.data_ptr(), L.dtype_code(qkv.dtype), n, num_heads, num_kv_heads,
                                    head_dim, positions.data_ptr(), slots.data_ptr(), rope_cos.data_ptr(),
                                    rope_sin.data_ptr(), rope_cos.shape[0], q_out.data_ptr(),
                                    pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), num_slots,
                                    L.ptr(status), L.stream_handle(qkv.device)))


def paged_attention(q, pool_k_layer, pool_v_layer, block_tables, ctx_lens, q_lens, q_offsets,
                    max_q_len: int, max_ctx: int, scale: float, out=None, workspace: Workspace | None = None,
                    status=None) -> torch.Tensor:
    """q [sum q_lens, nq, hd]; pools [num_blocks, bs, nkv, hd]; int32 tables/lengths."""
    lib = L.load()
    L.require_cuda(q, pool_k_layer, pool_v_layer, block_tables, ctx_lens, q_lens, q_offsets)
    _, nq, hd = q.shape
    num_blocks, bs, nkv, _ = pool_k_layer.shape
    B = ctx_lens.shape[0]
    for t in (block_tables, ctx_lens, q_lens, q_offsets):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("tables and lengths must be contiguous int32")
    if out is None:
        out = torch.empty_like(q)
    need = lib.kve_paged_attn_workspace_bytes(B, max_q_len, max_ctx, nq, nkv, hd)
    ws = (workspace or Workspace(q.device)).get(need) if need else None
    L.check(lib.kve_paged_verify_attn(
        q.data_ptr(), L.dtype_code(q.dtype), pool_k_layer.data_ptr(), pool_v_layer.data_ptr(),
        block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), q_lens.data_ptr(),
        q_offsets.data_ptr(), B, max_q_len, max_ctx, nq, nkv, hd, bs, num_blocks, scale, out.data_ptr(),
        L.ptr(ws), 0 if ws is None else ws.numel(), L.ptr(status), L.stream_handle(q.device)))
    return out


def gather_kv(pool_layer, block_table, length: int, status=None) -> torch.Tensor:
    """[nkv, length, hd] history of one sequence (pool_layer [num_blocks, bs, nkv, hd])."""
    lib = L.load()
    num_blocks, bs, nkv, hd = pool_layer.shape
    out = torch.empty(nkv, length, hd, dtype=pool_layer.dtype, device=pool_layer.device)
    L.check(lib.kve_gather_kv(pool_layer.data_ptr(), L.dtype_code(pool_layer.dtype), block_table.data_ptr(),
                              length, nkv, hd, bs, num_blocks, out.data_ptr(), L.ptr(status),
                              L.stream_handle(pool_layer.device)))
    return out


def embed(ids, table, out=None, status=None):
    lib = L.load()
    n = ids.shape[0]
    vocab, hidden = table.shape
    if out is None:
        out = torch.empty(n, hidden, dtype=table.dtype, device=table.device)
    L.check(lib.kve_embed(ids.data_ptr(), n, table.data_ptr(), L.dtype_code(table.dtype), hidden, vocab,
                          out.data_ptr(), L.ptr(status), L.stream_handle(table.device)))
    return out


def rmsnorm(x, weight, eps: float, row_index=None, out=None):
    lib = L.load()
    rows = x.shape[0] if row_index is None else row_index.shape[0]
    hidden = x.shape[1]
    if out is None:
        out = torch.empty(rows, hidden, dtype=x.dtype, device=x.device)
    L.check(lib.kve_rmsnorm(x.data_ptr(), L.dtype_code(x.dtype), weight.data_ptr(), rows, hidden, eps,
                            L.ptr(row_index), out.data_ptr(), L.stream_handle(x.device)))
    return out


def gemm(x, w, epilogue: int = L.EPI_STORE, bias=None, residual=None, out=None, out_dtype=None,
         workspace: Workspace | None = None, status=None, algo: int = L.GEMM_AUTO) -> torch.Tensor:
    lib = L.load()
    L.require_cuda(x, w)
    m, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k or x.dtype != w.dtype or not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("gemm: x [m,k] and w [n,k] must be contiguous and share a dtype")
    out_dtype = out_dtype or x.dtype
    n_out = n // 2 if epilogue == L.EPI_SILU_MUL else n
    if out is None:
        out = torch.empty(m, n_out, dtype=out_dtype, device=x.device)
    dc = L.dtype_code(x.dtype)
    need = lib.kve_gemm_workspace_bytes(m, n, k, dc)
    ws = (workspace or Workspace(x.device)).get(need) if need else None
    L.check(lib.kve_gemm_ex(x.data_ptr(), w.data_ptr(), dc, m, n, k, epilogue, L.ptr(bias), L.ptr(residual),
                            out.data_ptr(), L.dtype_code(out_dtype), L.ptr(ws), 0 if ws is None else ws.numel(),
                            L.ptr(status), algo, L.stream_handle(x.device)))
    return out


def spec_next_draft_plan(start_lens: torch.Tensor, last_tokens: torch.Tensor, n_blocks: torch.Tensor,
                         tables: torch.Tensor, block_size: int, k: int, rows: int, dump_block: int,
                         n_accepted: torch.Tensor, emitted: torch.Tensor, plan_out: torch.Tensor,
                         ids_out: torch.Tensor, verify_ids_out: torch.Tensor, status: torch.Tensor | None = None):
    """The next step's first draft pass planned on the device (kve_spec_next_draft_plan).
    start_lens, last_tokens, n_blocks [S], tables [S, width], n_accepted [S],
    emitted [S, k+1] (contiguous int32); writes plan_out (the packed ForwardPlan
    layout of `ForwardPlan.device_built(S, rows, width, ...)`), ids_out [rows * S]
    and verify_ids_out[s * (k+1)]."""
    lib = L.load()
    S = start_lens.numel()
    tensors = (start_lens, last_tokens, n_blocks, tables, n_accepted, emitted, plan_out, ids_out, verify_ids_out)
    L.require_cuda(*tensors)
    for t in tensors:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("spec_next_draft_plan takes contiguous int32 tensors")
    width = tables.numel() // max(S, 1)
    if tables.numel() != S * width or n_blocks.numel() != S or n_accepted.numel() < S or \
            emitted.numel() < S * (k + 1) or ids_out.numel() < rows * S or verify_ids_out.numel() < S * (k + 1) or \
            plan_out.numel() < 2 * rows * S + 4 * S + 1 + S * width:
        raise ValueError("spec_next_draft_plan: buffer sizes do not match")
    L.check(lib.kve_spec_next_draft_plan(start_lens.data_ptr(), last_tokens.data_ptr(), n_blocks.data_ptr(),
                                         tables.data_ptr(), S, width, block_size, k, rows, dump_block,
                                         n_accepted.data_ptr(), emitted.data_ptr(), plan_out.data_ptr(),
                                         ids_out.data_ptr(), verify_ids_out.data_ptr(), L.ptr(status),
                                         L.stream_handle(start_lens.device)))


# ------------------------------------------------ sampling, draft trees and the 8-bit cache
# These calls are a few microseconds of GPU work in a decode step: the C++ binding takes them
# where everything is as it should be, and what it leaves (it returns None) is checked and
# called here, where the errors are raised.
_I32, _F32, _U8, _E4M3 = torch.int32, torch.float32, torch.uint8, torch.float8_e4m3fn


def _refuse(name: str, rule: str) -> None:
    raise ValueError(f"{name}: {rule}")


def _dense(name: str, index: int, *tensors) -> None:
    """Every (tensor, dtype) is a contiguous tensor of that dtype on CUDA device `index`."""
    for at, (t, dtype) in enumerate(tensors):
        if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
            _refuse(name, f"tensor {at + 1} of {len(tensors)} checked together must be contiguous {dtype} on cuda:{index}, "
                          f"got {t.dtype} {list(t.shape)} with strides {t.stride()} on {t.device}")


def _device(t: torch.Tensor) -> int:
    index = t.get_device()
    if index < 0:
        L.require_cuda(t)
    return index


def _call(fn, index: int, *args) -> None:
    """fn(*args, stream) on the current stream of device `index`, which is made current if it is not."""
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, L.raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, L.raw_stream(index))
    if rc:
        L.check(rc)


def _status(name: str, index: int, status) -> int | None:
    if status is None:
        return None
    _dense(name, index, (status, _I32))
    if status.numel() < 1:
        _refuse(name, "status must have an element")
    return status.data_ptr()


def _space(name: str, index: int, workspace, device, need: int) -> torch.Tensor:
    buf = (workspace or Workspace(device)).get(need)
    _dense(name, index, (buf, _U8))  # a workspace of another device would be written there
    return buf


def _fp8_cache(name: str, index: int, k, v, k_scale, v_scale) -> None:
    _dense(name, index, (k, _E4M3), (v, _E4M3), (k_scale, _U8), (v_scale, _U8))
    shape = k.shape
    if v.shape != shape or k_scale.shape != shape[:-1] or v_scale.shape != shape[:-1]:
        _refuse(name, f"caches and scales of different shapes: {list(shape)}, {list(v.shape)}, {list(k_scale.shape)}, "
                      f"{list(v_scale.shape)}")


@lru_cache(maxsize=4096)
def _tree_attn_ws(*sizes: int) -> int:
    return L.load().kve_tree_attn_workspace_bytes(*sizes)


@lru_cache(maxsize=4096)
def _sample_ws(*sizes: int) -> int:
    return L.load().kve_sample_accept_workspace_bytes(*sizes)


@lru_cache(maxsize=4096)
def _tree_sample_ws(*sizes: int) -> int:
    return L.load().kve_tree_sample_accept_workspace_bytes(*sizes)


def tree_attention(q, pool_k_layer, pool_v_layer, block_tables, ctx_lens, q_lens, q_offsets, max_q_len: int, max_ctx: int,
                   scale: float, tree_mask=None, k_scale=None, v_scale=None, out=None, workspace: Workspace | None = None,
                   status=None) -> torch.Tensor:
    """Attention of drafted trees over a paged cache (kve_paged_tree_attn). Arguments as for
    `paged_attention`; tree_mask [sum q_lens, words] int32: bit t % 32 of word t / 32 of a row says
    whether it sees node t of its sequence (`tree_mask_words` builds it from parents; None: a
    chain); a row that sees nothing gets zeros, rows of `out` of no sequence are left as they are.
    bf16 queries also read an e4m3 cache, given its layer's k_scale and v_scale [num_blocks, bs,
    nkv] uint8."""
    r = L.fast().tree_attention(q, pool_k_layer, pool_v_layer, block_tables, ctx_lens, q_lens, q_offsets, max_q_len,
                                max_ctx, scale, tree_mask, k_scale, v_scale, out,
                                None if workspace is None else workspace.buf, status)
    if r is not None:
        if r.__class__ is int:
            L.check(r)
        return r
    lib = L.load()
    dev = _device(q)
    n, nq, hd = q.shape
    num_blocks, bs, nkv, pool_hd = pool_k_layer.shape
    B, width = block_tables.shape
    dtype = q.dtype
    code = L.dtype_code(dtype)
    if k_scale is None and v_scale is None:
        kv_code, ks, vs = code, None, None
        _dense("tree_attention", dev, (q, dtype), (pool_k_layer, dtype), (pool_v_layer, dtype), (block_tables, _I32),
               (ctx_lens, _I32), (q_lens, _I32), (q_offsets, _I32))
    else:
        if k_scale is None or v_scale is None:
            _refuse("tree_attention", "k_scale and v_scale go together")
        kv_code, ks, vs = L.KVE_FP8_E4M3, k_scale.data_ptr(), v_scale.data_ptr()
        _dense("tree_attention", dev, (q, torch.bfloat16), (block_tables, _I32), (ctx_lens, _I32), (q_lens, _I32),
               (q_offsets, _I32))
        _fp8_cache("tree_attention", dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    if pool_hd != hd or pool_v_layer.shape != pool_k_layer.shape:
        _refuse("tree_attention", f"head_dim {hd} of q, caches {list(pool_k_layer.shape)} and {list(pool_v_layer.shape)}")
    if ctx_lens.numel() != B or q_lens.numel() != B or q_offsets.numel() < B:
        _refuse("tree_attention", "one block table row, length and offset per sequence")
    mask, words = None, 0
    if tree_mask is not None:
        _dense("tree_attention", dev, (tree_mask, _I32))
        rows, words = tree_mask.shape
        if rows != n:
            _refuse("tree_attention", "one tree_mask row per row of q")
        mask = tree_mask.data_ptr()
    if out is None:
        out = torch.empty_like(q)
    else:
        _dense("tree_attention", dev, (out, dtype))
        if out.shape != q.shape:
            _refuse("tree_attention", "out has the shape of q")
    need = _tree_attn_ws(B, max_q_len, max_ctx, nq, nkv, hd)
    ws, ws_bytes = None, 0
    if need:
        buf = _space("tree_attention", dev, workspace, q.device, need)
        ws, ws_bytes = buf.data_ptr(), buf.numel()
    _call(lib.kve_paged_tree_attn, dev, q.data_ptr(), code, pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), kv_code, ks, vs,
          block_tables.data_ptr(), width, ctx_lens.data_ptr(), q_lens.data_ptr(), q_offsets.data_ptr(), mask, words, B, n,
          max_q_len, max_ctx, nq, nkv, hd, bs, num_blocks, scale, out.data_ptr(), ws, ws_bytes,
          _status("tree_attention", dev, status))
    return out


def tree_mask_words(parents: list[list[int]], max_q_len: int | None = None) -> torch.Tensor:
    """Host mask rows for `tree_attention`: parents[b][i] is the parent of node i of sequence b's
    tree (-1: none; a parent comes before its children). A node sees itself and its ancestors.
    Returns int32 [sum of nodes, ceil(max_q_len / 32)]."""
    longest = max((len(t) for t in parents), default=0)
    words = max(1, -(-max(longest, max_q_len or 0) // 32))
    rows = []
    for t in parents:
        seen: list[int] = []
        for i, p in enumerate(t):
            if not -1 <= p < i:
                raise ValueError(f"tree_mask_words: node {i} has parent {p}")
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        rows += seen
    flat = b"".join(bits.to_bytes(4 * words, "little") for bits in rows)
    return torch.frombuffer(bytearray(flat), dtype=torch.int32).view(-1, words) if rows else \
        torch.zeros(0, words, dtype=torch.int32)


def qkv_rope_append_fp8(qkv, positions, slots, rope_cos, rope_sin, q_out, pool_k_layer, pool_v_layer, k_scale, v_scale,
                        num_heads, num_kv_heads, head_dim, status=None) -> None:
    """`qkv_rope_append` into an e4m3 cache (pools [num_blocks, bs, nkv, hd] float8_e4m3fn, scales
    [num_blocks, bs, nkv] uint8): q rotated into q_out, K rotated and quantised, V quantised."""
    r = L.fast().qkv_rope_append_fp8(qkv, positions, slots, rope_cos, rope_sin, q_out, pool_k_layer, pool_v_layer,
                                     k_scale, v_scale, num_heads, num_kv_heads, head_dim, status)
    if r is not None:
        if r.__class__ is int:
            L.check(r)
        return
    lib = L.load()
    name = "qkv_rope_append_fp8"
    dev, dtype = _device(qkv), qkv.dtype
    n, width = qkv.shape
    _dense(name, dev, (qkv, dtype), (positions, _I32), (slots, _I32), (rope_cos, _F32), (rope_sin, _F32), (q_out, dtype))
    _fp8_cache(name, dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    num_blocks, bs, nkv, hd = pool_k_layer.shape
    rope_len, half = rope_cos.shape
    if width != (num_heads + 2 * num_kv_heads) * head_dim or nkv != num_kv_heads or hd != head_dim or \
            positions.numel() != n or slots.numel() != n or half * 2 != hd or rope_sin.shape != rope_cos.shape or \
            q_out.numel() != n * num_heads * head_dim:
        _refuse(name, f"shapes do not fit {num_heads}/{num_kv_heads} heads of {head_dim}: qkv {list(qkv.shape)}, positions "
                      f"{list(positions.shape)}, slots {list(slots.shape)}, tables {list(rope_cos.shape)} "
                      f"{list(rope_sin.shape)}, q_out {list(q_out.shape)}, cache {list(pool_k_layer.shape)}")
    _call(lib.kve_qkv_rope_append_fp8, dev, qkv.data_ptr(), L.dtype_code(dtype), n, num_heads, num_kv_heads, head_dim,
          positions.data_ptr(), slots.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(), rope_len, q_out.data_ptr(),
          pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), num_blocks * bs,
          _status(name, dev, status))


def kv_append_fp8(k_new, v_new, slot_ids, pool_k_layer, pool_v_layer, k_scale, v_scale, status=None) -> None:
    """`kv_append` into an e4m3 cache: rows [n, nkv, hd] quantised, each with its own power of two."""
    lib = L.load()
    dev, dtype = _device(k_new), k_new.dtype
    n, nkv, hd = k_new.shape
    _dense("kv_append_fp8", dev, (k_new, dtype), (v_new, dtype), (slot_ids, torch.int64))
    _fp8_cache("kv_append_fp8", dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    num_blocks, bs, *heads = pool_k_layer.shape
    if heads != [nkv, hd] or v_new.shape != k_new.shape or slot_ids.numel() != n:
        _refuse("kv_append_fp8", f"rows {list(k_new.shape)} and {list(v_new.shape)}, {slot_ids.numel()} slots, cache "
                                 f"{list(pool_k_layer.shape)}")
    _call(lib.kve_kv_append_fp8, dev, k_new.data_ptr(), v_new.data_ptr(), L.dtype_code(dtype), slot_ids.data_ptr(), n, nkv,
          hd, pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), num_blocks * bs,
          _status("kv_append_fp8", dev, status))


def kv_read_fp8(pool_k_layer, pool_v_layer, k_scale, v_scale, slot_ids, dtype: torch.dtype = torch.bfloat16, out=None,
                status=None):
    """Rows of an e4m3 cache as the values they stand for: (k, v), each [n, nkv, hd] in `dtype`, of
    the flat slots slot_ids [n] int64. `out` may give the two."""
    if out is None and (dtype is torch.bfloat16 or dtype is _F32):
        r = L.fast().kv_read_fp8(pool_k_layer, pool_v_layer, k_scale, v_scale, slot_ids, int(dtype is torch.bfloat16), status)
        if r is not None:
            if r.__class__ is int:
                L.check(r)
            return r
    lib = L.load()
    dev = _device(pool_k_layer)
    num_blocks, bs, nkv, hd = pool_k_layer.shape
    _fp8_cache("kv_read_fp8", dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    _dense("kv_read_fp8", dev, (slot_ids, torch.int64))
    (n,) = slot_ids.shape
    if out is None:
        k = torch.empty(n, nkv, hd, dtype=dtype, device=pool_k_layer.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        _dense("kv_read_fp8", dev, (k, dtype), (v, dtype))
        if k.shape != (n, nkv, hd) or v.shape != (n, nkv, hd):
            _refuse("kv_read_fp8", f"out must be two tensors [{n}, {nkv}, {hd}]")
    _call(lib.kve_kv_read_fp8, dev, pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
          slot_ids.data_ptr(), n, nkv, hd, num_blocks * bs, L.dtype_code(dtype), k.data_ptr(), v.data_ptr(),
          _status("kv_read_fp8", dev, status))
    return k, v


def _rows(name: str, what: str, index: int, t: torch.Tensor, dtype, rows: int, cols: int) -> int:
    """The row stride of a [rows, cols] matrix with unit column stride on device `index`."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != (rows, cols):
        _refuse(name, f"{what} must be {dtype} [{rows}, {cols}] on cuda:{index}, got {t.dtype} {list(t.shape)} on {t.device}")
    if t.is_contiguous():
        return cols
    stride, unit = t.stride()
    if (cols > 1 and unit != 1) or (rows > 1 and stride < cols):
        _refuse(name, f"{what} needs unit column stride and rows apart, got strides {t.stride()}")
    return max(stride, cols)


def sample_accept(logits: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor, gumbel: torch.Tensor,
                  temperature: torch.Tensor, draft_logits: torch.Tensor | None = None,
                  workspace: Workspace | None = None, status: torch.Tensor | None = None, out=None):
    """`greedy_accept` for sampling (kve_sample_accept): logits [B, k+1, V], drafts [B, k] int32 (any
    strides), uniforms [B, k] in [0, 1), gumbel [B, V] noise -log(-log u), temperature [B]
    (0: greedy), draft_logits [B, k, V] (None: drafts without a distribution) ->
    (n_accepted [B], emitted [B, k+1], logprobs [B, k+1]). `out` may give the three."""
    if out is None:
        r = L.fast().sample_accept(logits, drafts, uniforms, gumbel, temperature, draft_logits,
                                   None if workspace is None else workspace.buf, status)
        if r is not None:
            if r.__class__ is int:
                L.check(r)
            return r
    lib = L.load()
    name = "sample_accept"
    dev, dtype = _device(logits), logits.dtype
    B, kp1, V = logits.shape
    k = kp1 - 1
    if drafts.dtype is not _I32 or drafts.shape != (B, k) or drafts.get_device() != dev:
        _refuse(name, f"drafts must be int32 [{B}, {k}] on cuda:{dev}")
    stride = V
    if not logits.is_contiguous():
        sb, stride, unit = logits.stride()
        if (V > 1 and unit != 1) or (B > 1 and sb != kp1 * stride) or stride < V:
            _refuse(name, "logits rows must be evenly strided with unit column stride")
    usb = _rows(name, "uniforms", dev, uniforms, _F32, B, k)
    gs = _rows(name, "gumbel", dev, gumbel, _F32, B, V)
    _dense(name, dev, (temperature, _F32))
    if temperature.numel() != B:
        _refuse(name, f"temperature must have {B} elements")
    dl, dlb, dlj = None, 0, 0
    if draft_logits is not None:
        dlb, dlj, unit = draft_logits.stride()
        if draft_logits.dtype is not dtype or draft_logits.shape != (B, k, V) or draft_logits.get_device() != dev or \
                (V > 1 and unit != 1):
            _refuse(name, f"draft_logits must be {dtype} [{B}, {k}, {V}] on cuda:{dev} with unit column stride")
        dl = draft_logits.data_ptr()
    if out is None:
        device = logits.device
        n_acc = torch.empty(B, dtype=_I32, device=device)
        emitted = torch.empty(B, kp1, dtype=_I32, device=device)
        logprobs = torch.empty(B, kp1, dtype=_F32, device=device)
    else:
        n_acc, emitted, logprobs = out
        _dense(name, dev, (n_acc, _I32), (emitted, _I32), (logprobs, _F32))
        if n_acc.numel() != B or emitted.shape != (B, kp1) or logprobs.shape != (B, kp1):
            _refuse(name, f"out must be [{B}], [{B}, {kp1}] and [{B}, {kp1}]")
    ws = _space(name, dev, workspace, logits.device, _sample_ws(B, k, V, int(dl is not None)))
    dsb, dsj = drafts.stride()
    _call(lib.kve_sample_accept, dev, logits.data_ptr(), L.dtype_code(dtype), stride, dl, dlb, dlj, drafts.data_ptr(), dsb,
          dsj, uniforms.data_ptr(), usb, gumbel.data_ptr(), gs, temperature.data_ptr(), B, k, V, n_acc.data_ptr(),
          emitted.data_ptr(), logprobs.data_ptr(), ws.data_ptr(), ws.numel(), _status(name, dev, status))
    return n_acc, emitted, logprobs


def tree_sample_accept(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, q_lens: torch.Tensor,
                       q_offsets: torch.Tensor, max_q_len: int, uniforms: torch.Tensor, gumbel: torch.Tensor,
                       temperature: torch.Tensor, workspace: Workspace | None = None,
                       status: torch.Tensor | None = None, out=None):
    """Verification of draft trees by sampling (kve_tree_sample_accept): logits [N, V] and tokens,
    parents (int32), uniforms [N] of the trees' nodes, sequence b's at rows q_offsets[b] .. +
    q_lens[b] (parents within the tree, node 0 its root; offsets ascend, rows are not shared); gumbel
    [B, V], temperature [B] -> (n_accepted [B], path, emitted, logprobs [B, max_q_len]). A sequence
    without nodes gets n_accepted -1, and its rows of the other three are not written. `out` may
    give the four."""
    if out is None:
        r = L.fast().tree_sample_accept(logits, tokens, parents, q_lens, q_offsets, max_q_len, uniforms, gumbel,
                                        temperature, None if workspace is None else workspace.buf, status)
        if r is not None:
            if r.__class__ is int:
                L.check(r)
            return r
    lib = L.load()
    name = "tree_sample_accept"
    dev, dtype = _device(logits), logits.dtype
    N, V = logits.shape
    B = q_lens.numel()
    stride = _rows(name, "logits", dev, logits, dtype, N, V)
    gs = _rows(name, "gumbel", dev, gumbel, _F32, B, V)
    _dense(name, dev, (tokens, _I32), (parents, _I32), (uniforms, _F32), (q_lens, _I32), (q_offsets, _I32),
           (temperature, _F32))
    if tokens.numel() != N or parents.numel() != N or uniforms.numel() != N or q_offsets.numel() < B or \
            temperature.numel() != B:
        _refuse(name, f"{N} rows need as many tokens, parents and uniforms, {B} sequences as many offsets and temperatures")
    if out is None:
        device = logits.device
        n_acc = torch.empty(B, dtype=_I32, device=device)
        path = torch.empty(B, max_q_len, dtype=_I32, device=device)
        emitted = torch.empty_like(path)
        logprobs = torch.empty(B, max_q_len, dtype=_F32, device=device)
    else:
        n_acc, path, emitted, logprobs = out
        _dense(name, dev, (n_acc, _I32), (path, _I32), (emitted, _I32), (logprobs, _F32))
        shape = (B, max_q_len)
        if n_acc.numel() != B or path.shape != shape or emitted.shape != shape or logprobs.shape != shape:
            _refuse(name, f"out must be [{B}] and three times [{B}, {max_q_len}]")
    ws = _space(name, dev, workspace, logits.device, _tree_sample_ws(N, V))
    _call(lib.kve_tree_sample_accept, dev, logits.data_ptr(), L.dtype_code(dtype), stride, tokens.data_ptr(),
          parents.data_ptr(), q_lens.data_ptr(), q_offsets.data_ptr(), uniforms.data_ptr(), gumbel.data_ptr(), gs,
          temperature.data_ptr(), B, N, max_q_len, V, n_acc.data_ptr(), path.data_ptr(), emitted.data_ptr(),
          logprobs.data_ptr(), ws.data_ptr(), ws.numel(), _status(name, dev, status))
    return n_acc, path, emitted, logprobs


def kv_commit_path(pool_k, pool_v, block_tables, start_lens, path, n_accepted, k_scale=None, v_scale=None,
                   status=None) -> None:
    """Move the accepted path's K/V together in every layer (kve_kv_commit_path): for j = 1 ..
    n_accepted[b], position start_lens[b] + path[b, j] -> start_lens[b] + j. pools [L, num_blocks, bs,
    nkv, hd] (an e4m3 cache with its scales [L, num_blocks, bs, nkv]); path [B, P] and n_accepted
    [B] int32 as `tree_sample_accept` gives them; start_lens [B] the positions of the trees' node 0."""
    r = L.fast().kv_commit_path(pool_k, pool_v, block_tables, start_lens, path, n_accepted, k_scale, v_scale, status)
    if r is not None:
        if r.__class__ is int:
            L.check(r)
        return
    lib = L.load()
    dev = _device(pool_k)
    layers, num_blocks, bs, nkv, hd = pool_k.shape
    B, width = block_tables.shape
    path_rows, path_width = path.shape
    if k_scale is None and v_scale is None:
        code, ks, vs = L.dtype_code(pool_k.dtype), None, None
        _dense("kv_commit_path", dev, (pool_k, pool_k.dtype), (pool_v, pool_k.dtype), (block_tables, _I32), (start_lens, _I32),
               (path, _I32), (n_accepted, _I32))
        if pool_v.shape != pool_k.shape:
            _refuse("kv_commit_path", f"caches of different shapes: {list(pool_k.shape)}, {list(pool_v.shape)}")
    else:
        if k_scale is None or v_scale is None:
            _refuse("kv_commit_path", "k_scale and v_scale go together")
        code, ks, vs = L.KVE_FP8_E4M3, k_scale.data_ptr(), v_scale.data_ptr()
        _fp8_cache("kv_commit_path", dev, pool_k, pool_v, k_scale, v_scale)
        _dense("kv_commit_path", dev, (block_tables, _I32), (start_lens, _I32), (path, _I32), (n_accepted, _I32))
    if path_rows != B or start_lens.numel() != B or n_accepted.numel() != B:
        _refuse("kv_commit_path", "one block table row, path row, start and count per sequence")
    _call(lib.kve_kv_commit_path, dev, pool_k.data_ptr(), pool_v.data_ptr(), code, ks, vs, layers, num_blocks, bs, nkv, hd,
          block_tables.data_ptr(), width, start_lens.data_ptr(), path.data_ptr(), path_width, n_accepted.data_ptr(), B,
          _status("kv_commit_path", dev, status))
