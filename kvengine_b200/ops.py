"""Torch-tensor wrappers over the C ABI, one per kernel entry point.

Each wrapper checks shapes, dtypes and devices on the host, then launches on
the current CUDA stream. Workspaces are plain zero-filled uint8 tensors the
caller keeps (the kernels leave them zeroed).
"""

from __future__ import annotations

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
def _like(name: str, dev: torch.device, **tensors) -> None:
    """Every given (tensor, dtype, shape) is a contiguous tensor of that dtype and shape on `dev`
    (a shape of None: any)."""
    for what, (t, dtype, shape) in tensors.items():
        if t.dtype != dtype or t.device != dev or not t.is_contiguous() or (shape is not None and t.shape != shape):
            raise ValueError(f"{name}: {what} must be a contiguous {dtype} tensor"
                             f"{'' if shape is None else ' ' + str(list(shape))} on {dev}, got {t.dtype} {list(t.shape)} "
                             f"with strides {t.stride()} on {t.device}")


def _call(fn, dev: torch.device, *args) -> None:
    """fn(*args, stream) on the current stream of `dev`, which is made current if it is not."""
    if dev.index == torch.cuda.current_device():
        L.check(fn(*args, L.stream_handle(dev)))
    else:
        with torch.cuda.device(dev):
            L.check(fn(*args, L.stream_handle(dev)))


def _fp8_cache(name: str, dev, k, v, k_scale, v_scale) -> None:
    _like(name, dev, pool_k=(k, torch.float8_e4m3fn, None), pool_v=(v, torch.float8_e4m3fn, k.shape),
          k_scale=(k_scale, torch.uint8, k.shape[:-1]), v_scale=(v_scale, torch.uint8, k.shape[:-1]))


def tree_attention(q, pool_k_layer, pool_v_layer, block_tables, ctx_lens, q_lens, q_offsets, max_q_len: int, max_ctx: int,
                   scale: float, tree_mask=None, k_scale=None, v_scale=None, out=None, workspace: Workspace | None = None,
                   status=None) -> torch.Tensor:
    """Attention of drafted trees over a paged cache (kve_paged_tree_attn). Arguments as for
    `paged_attention`; tree_mask [sum q_lens, words] int32: bit t % 32 of word t / 32 of a row says
    whether it sees node t of its sequence (`tree_mask_words` builds it from parents; None: a
    chain); a row that sees nothing gets zeros. bf16 queries also read an e4m3 cache, given
    its layer's k_scale and v_scale [num_blocks, bs, nkv] uint8."""
    lib = L.load()
    L.require_cuda(q)
    dev = q.device
    n, nq, hd = q.shape
    num_blocks, bs, nkv, pool_hd = pool_k_layer.shape
    B = ctx_lens.shape[0]
    if pool_hd != hd:
        raise ValueError(f"tree_attention: head_dim {hd} of q, {pool_hd} of the cache")
    if k_scale is None and v_scale is None:
        kv_code = L.dtype_code(q.dtype)
        _like("tree_attention", dev, q=(q, q.dtype, None), pool_k=(pool_k_layer, q.dtype, None),
              pool_v=(pool_v_layer, q.dtype, pool_k_layer.shape))
    else:
        kv_code = L.KVE_FP8_E4M3
        if k_scale is None or v_scale is None:
            raise ValueError("tree_attention: k_scale and v_scale go together")
        _like("tree_attention", dev, q=(q, torch.bfloat16, None))
        _fp8_cache("tree_attention", dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    i32 = torch.int32
    _like("tree_attention", dev, block_tables=(block_tables, i32, None), ctx_lens=(ctx_lens, i32, None),
          q_lens=(q_lens, i32, ctx_lens.shape), q_offsets=(q_offsets, i32, None))
    if block_tables.dim() != 2 or block_tables.shape[0] != B or q_offsets.shape[0] < B:
        raise ValueError("tree_attention: one block table row, length and offset per sequence")
    words = 0
    if tree_mask is not None:
        _like("tree_attention", dev, tree_mask=(tree_mask, i32, None))
        if tree_mask.dim() != 2 or tree_mask.shape[0] != n:
            raise ValueError("tree_attention: one tree_mask row per row of q")
        words = tree_mask.shape[1]
    if out is None:
        out = torch.empty_like(q)
    else:
        _like("tree_attention", dev, out=(out, q.dtype, q.shape))
    need = lib.kve_tree_attn_workspace_bytes(B, max_q_len, max_ctx, nq, nkv, hd)
    ws, ws_bytes = None, 0
    if need:
        buf = (workspace or Workspace(dev)).get(need)
        ws, ws_bytes = buf.data_ptr(), buf.numel()
    _call(lib.kve_paged_tree_attn, dev, q.data_ptr(), L.dtype_code(q.dtype), pool_k_layer.data_ptr(), pool_v_layer.data_ptr(),
          kv_code, L.ptr(k_scale), L.ptr(v_scale), block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(),
          q_lens.data_ptr(), q_offsets.data_ptr(), L.ptr(tree_mask), words, B, max_q_len, max_ctx, nq, nkv, hd, bs,
          num_blocks, scale, out.data_ptr(), ws, ws_bytes, L.ptr(status))
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
    lib = L.load()
    L.require_cuda(qkv)
    dev, n = qkv.device, qkv.shape[0]
    name = "qkv_rope_append_fp8"
    _like(name, dev, qkv=(qkv, qkv.dtype, (n, (num_heads + 2 * num_kv_heads) * head_dim)),
          positions=(positions, torch.int32, (n,)), slots=(slots, torch.int32, (n,)),
          rope_cos=(rope_cos, torch.float32, (rope_cos.shape[0], head_dim // 2)),
          rope_sin=(rope_sin, torch.float32, rope_cos.shape))
    if q_out.numel() != n * num_heads * head_dim:
        raise ValueError(f"{name}: q_out must have n_tokens x num_heads x head_dim elements")
    _like(name, dev, q_out=(q_out, qkv.dtype, None))
    _fp8_cache(name, dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    if pool_k_layer.shape[2:] != (num_kv_heads, head_dim):
        raise ValueError(f"{name}: the cache has heads {list(pool_k_layer.shape[2:])}")
    _call(lib.kve_qkv_rope_append_fp8, dev, qkv.data_ptr(), L.dtype_code(qkv.dtype), n, num_heads, num_kv_heads, head_dim,
          positions.data_ptr(), slots.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(), rope_cos.shape[0],
          q_out.data_ptr(), pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
          pool_k_layer.shape[0] * pool_k_layer.shape[1], L.ptr(status))


def kv_append_fp8(k_new, v_new, slot_ids, pool_k_layer, pool_v_layer, k_scale, v_scale, status=None) -> None:
    """`kv_append` into an e4m3 cache: rows [n, nkv, hd] quantised, each with its own power of two."""
    lib = L.load()
    L.require_cuda(k_new)
    dev = k_new.device
    n, nkv, hd = k_new.shape
    _like("kv_append_fp8", dev, k_new=(k_new, k_new.dtype, None), v_new=(v_new, k_new.dtype, k_new.shape),
          slot_ids=(slot_ids, torch.int64, (n,)))
    _fp8_cache("kv_append_fp8", dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    if pool_k_layer.shape[2:] != (nkv, hd):
        raise ValueError(f"kv_append_fp8: the cache has heads {list(pool_k_layer.shape[2:])}")
    _call(lib.kve_kv_append_fp8, dev, k_new.data_ptr(), v_new.data_ptr(), L.dtype_code(k_new.dtype), slot_ids.data_ptr(), n,
          nkv, hd, pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
          pool_k_layer.shape[0] * pool_k_layer.shape[1], L.ptr(status))


def kv_read_fp8(pool_k_layer, pool_v_layer, k_scale, v_scale, slot_ids, dtype: torch.dtype = torch.bfloat16, out=None,
                status=None):
    """Rows of an e4m3 cache as the values they stand for: (k, v), each [n, nkv, hd] in `dtype`, of
    the flat slots slot_ids [n] int64. `out` may give the two."""
    lib = L.load()
    L.require_cuda(pool_k_layer)
    dev = pool_k_layer.device
    num_blocks, bs, nkv, hd = pool_k_layer.shape
    n = slot_ids.shape[0]
    _fp8_cache("kv_read_fp8", dev, pool_k_layer, pool_v_layer, k_scale, v_scale)
    _like("kv_read_fp8", dev, slot_ids=(slot_ids, torch.int64, (n,)))
    if out is None:
        k = torch.empty(n, nkv, hd, dtype=dtype, device=dev)
        v = torch.empty_like(k)
    else:
        k, v = out
        _like("kv_read_fp8", dev, k_out=(k, dtype, (n, nkv, hd)), v_out=(v, dtype, (n, nkv, hd)))
    _call(lib.kve_kv_read_fp8, dev, pool_k_layer.data_ptr(), pool_v_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
          slot_ids.data_ptr(), n, nkv, hd, num_blocks * bs, L.dtype_code(dtype), k.data_ptr(), v.data_ptr(), L.ptr(status))
    return k, v


def _noise(name: str, dev, gumbel, temperature, B: int, V: int) -> None:
    _like(name, dev, temperature=(temperature, torch.float32, (B,)))
    if gumbel.dtype != torch.float32 or gumbel.shape != (B, V) or gumbel.device != dev or \
            (V > 1 and gumbel.stride(1) != 1) or (B > 1 and gumbel.stride(0) < V):
        raise ValueError(f"{name}: gumbel must be float32 [{B}, {V}] on {dev} with unit column stride")


def sample_accept(logits: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor, gumbel: torch.Tensor,
                  temperature: torch.Tensor, draft_logits: torch.Tensor | None = None,
                  workspace: Workspace | None = None, status: torch.Tensor | None = None, out=None):
    """`greedy_accept` for sampling (kve_sample_accept): logits [B, k+1, V], drafts [B, k] int32 (any
    strides), uniforms [B, k] in [0, 1), gumbel [B, V] noise -log(-log u), temperature [B]
    (0: greedy), draft_logits [B, k, V] (None: drafts without a distribution) ->
    (n_accepted [B], emitted [B, k+1], logprobs [B, k+1]). `out` may give the three."""
    lib = L.load()
    L.require_cuda(logits)
    dev = logits.device
    B, kp1, V = logits.shape
    k = kp1 - 1
    if drafts.dtype != torch.int32 or drafts.shape != (B, k) or drafts.device != dev:
        raise ValueError(f"sample_accept: drafts must be int32 [{B}, {k}] on {dev}")
    if logits.stride(2) != 1 or (B > 1 and logits.stride(0) != kp1 * logits.stride(1)):
        raise ValueError("sample_accept: logits rows must be evenly strided with unit column stride")
    if uniforms.dtype != torch.float32 or uniforms.shape != (B, k) or uniforms.device != dev or \
            (k > 1 and uniforms.stride(1) != 1) or (B > 1 and uniforms.stride(0) < k):
        raise ValueError(f"sample_accept: uniforms must be float32 [{B}, {k}] on {dev} with unit column stride")
    _noise("sample_accept", dev, gumbel, temperature, B, V)
    dsb = dsj = 0
    if draft_logits is not None:
        if draft_logits.dtype != logits.dtype or draft_logits.shape != (B, k, V) or draft_logits.device != dev or \
                (V > 1 and draft_logits.stride(2) != 1):
            raise ValueError(f"sample_accept: draft_logits must be {logits.dtype} [{B}, {k}, {V}] on {dev} with unit column "
                             "stride")
        dsb, dsj = draft_logits.stride(0), draft_logits.stride(1)
    if out is None:
        n_acc = torch.empty(B, dtype=torch.int32, device=dev)
        emitted = torch.empty(B, kp1, dtype=torch.int32, device=dev)
        logprobs = torch.empty(B, kp1, dtype=torch.float32, device=dev)
    else:
        n_acc, emitted, logprobs = out
        _like("sample_accept", dev, n_accepted=(n_acc, torch.int32, (B,)), emitted=(emitted, torch.int32, (B, kp1)),
              logprobs=(logprobs, torch.float32, (B, kp1)))
    ws = (workspace or Workspace(dev)).get(lib.kve_sample_accept_workspace_bytes(B, k, V, draft_logits is not None))
    _call(lib.kve_sample_accept, dev, logits.data_ptr(), L.dtype_code(logits.dtype), max(logits.stride(1), V),
          L.ptr(draft_logits), dsb, dsj, drafts.data_ptr(), drafts.stride(0), drafts.stride(1), uniforms.data_ptr(),
          max(uniforms.stride(0), k), gumbel.data_ptr(), max(gumbel.stride(0), V), temperature.data_ptr(), B, k, V,
          n_acc.data_ptr(), emitted.data_ptr(), logprobs.data_ptr(), ws.data_ptr(), ws.numel(), L.ptr(status))
    return n_acc, emitted, logprobs


def tree_sample_accept(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, q_lens: torch.Tensor,
                       q_offsets: torch.Tensor, max_q_len: int, uniforms: torch.Tensor, gumbel: torch.Tensor,
                       temperature: torch.Tensor, workspace: Workspace | None = None,
                       status: torch.Tensor | None = None, out=None):
    """Verification of draft trees by sampling (kve_tree_sample_accept): logits [N, V] and tokens,
    parents (int32), uniforms [N] of the trees' nodes, sequence b's at rows q_offsets[b] .. +
    q_lens[b] (parents within the tree, node 0 its root); gumbel [B, V], temperature [B] ->
    (n_accepted [B], path, emitted, logprobs [B, max_q_len]). `out` may give the four."""
    lib = L.load()
    L.require_cuda(logits)
    dev = logits.device
    N, V = logits.shape
    B = q_lens.shape[0]
    name = "tree_sample_accept"
    if (V > 1 and logits.stride(1) != 1) or (N > 1 and logits.stride(0) < V):
        raise ValueError(f"{name}: logits needs unit column stride")
    i32, f32 = torch.int32, torch.float32
    _like(name, dev, tokens=(tokens, i32, (N,)), parents=(parents, i32, (N,)), uniforms=(uniforms, f32, (N,)),
          q_lens=(q_lens, i32, (B,)), q_offsets=(q_offsets, i32, None))
    if q_offsets.shape[0] < B:
        raise ValueError(f"{name}: one offset per sequence")
    _noise(name, dev, gumbel, temperature, B, V)
    if out is None:
        n_acc = torch.empty(B, dtype=i32, device=dev)
        path = torch.empty(B, max_q_len, dtype=i32, device=dev)
        emitted = torch.empty_like(path)
        logprobs = torch.empty(B, max_q_len, dtype=f32, device=dev)
    else:
        n_acc, path, emitted, logprobs = out
        shape = (B, max_q_len)
        _like(name, dev, n_accepted=(n_acc, i32, (B,)), path=(path, i32, shape), emitted=(emitted, i32, shape),
              logprobs=(logprobs, f32, shape))
    ws = (workspace or Workspace(dev)).get(lib.kve_tree_sample_accept_workspace_bytes(N, V))
    _call(lib.kve_tree_sample_accept, dev, logits.data_ptr(), L.dtype_code(logits.dtype), max(logits.stride(0), V),
          tokens.data_ptr(), parents.data_ptr(), q_lens.data_ptr(), q_offsets.data_ptr(), uniforms.data_ptr(),
          gumbel.data_ptr(), max(gumbel.stride(0), V), temperature.data_ptr(), B, N, max_q_len, V, n_acc.data_ptr(),
          path.data_ptr(), emitted.data_ptr(), logprobs.data_ptr(), ws.data_ptr(), ws.numel(), L.ptr(status))
    return n_acc, path, emitted, logprobs


def kv_commit_path(pool_k, pool_v, block_tables, start_lens, path, n_accepted, k_scale=None, v_scale=None,
                   status=None) -> None:
    """Move the accepted path's K/V together in every layer (kve_kv_commit_path): for j = 1 ..
    n_accepted[b], position start_lens[b] + path[b, j] -> start_lens[b] + j. pools [L, num_blocks, bs,
    nkv, hd] (an e4m3 cache with its scales [L, num_blocks, bs, nkv]); path [B, P] and n_accepted
    [B] int32 as `tree_sample_accept` gives them; start_lens [B] the positions of the trees' node 0."""
    lib = L.load()
    L.require_cuda(pool_k)
    dev = pool_k.device
    layers, num_blocks, bs, nkv, hd = pool_k.shape
    B, i32 = start_lens.shape[0], torch.int32
    if k_scale is None and v_scale is None:
        code = L.dtype_code(pool_k.dtype)
        _like("kv_commit_path", dev, pool_k=(pool_k, pool_k.dtype, None), pool_v=(pool_v, pool_k.dtype, pool_k.shape))
    else:
        code = L.KVE_FP8_E4M3
        if k_scale is None or v_scale is None:
            raise ValueError("kv_commit_path: k_scale and v_scale go together")
        _fp8_cache("kv_commit_path", dev, pool_k, pool_v, k_scale, v_scale)
    _like("kv_commit_path", dev, block_tables=(block_tables, i32, None), start_lens=(start_lens, i32, None),
          path=(path, i32, None), n_accepted=(n_accepted, i32, (B,)))
    if block_tables.dim() != 2 or block_tables.shape[0] != B or path.dim() != 2 or path.shape[0] != B:
        raise ValueError("kv_commit_path: one block table row and one path row per sequence")
    _call(lib.kve_kv_commit_path, dev, pool_k.data_ptr(), pool_v.data_ptr(), code, L.ptr(k_scale), L.ptr(v_scale), layers,
          num_blocks, bs, nkv, hd, block_tables.data_ptr(), block_tables.shape[1], start_lens.data_ptr(), path.data_ptr(),
          path.shape[1], n_accepted.data_ptr(), B, L.ptr(status))
