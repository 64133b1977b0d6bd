"""Calls into the kernel C ABI with torch CUDA tensors.

torch only provides device memory and the current stream here; every
computation is one of the library's kernels. Used by the parity tests and
the benchmark.
"""

import ctypes

import torch

from ._lib import P_i64, Epilogue, L2Prefetch, Q8CacheStruct, Q8Plane, check, load

ACT = {"none": 0, "relu": 1, "gelu": 2}


def _s(stream=None):
    return ctypes.c_void_p((stream or torch.cuda.current_stream()).cuda_stream)


def _p(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def embed(ids, table, seq, id_offset=0, status=None):
    hidden = table.shape[1]
    out = torch.zeros(seq, hidden, dtype=torch.float32, device=table.device)
    check(load().accel_b200_embed(_p(ids), id_offset, _p(table), _p(out), seq, hidden, table.shape[0], _p(status), _s()))
    return out


def rmsnorm(x, w, rows, dim, eps, row_offset=0):
    y = torch.zeros(rows, dim, dtype=torch.float32, device=x.device)
    check(load().accel_b200_rmsnorm(_p(x), _p(w), _p(y), rows, dim, eps, row_offset, _s()))
    return y


def rope(states, cos_t, sin_t, seq, n_heads, head_dim, position):
    check(load().accel_b200_rope(_p(states), _p(cos_t), _p(sin_t), seq, n_heads, head_dim, position, _s()))
    return states


def append_cache(src, cache, seq, position, n_heads, head_dim):
    check(load().accel_b200_append_cache(_p(src), _p(cache), seq, position, n_heads, head_dim, _s()))
    return cache


def attention(q, k, v, seq, position, heads, kv_heads, head_dim):
    out = torch.zeros(seq, heads, head_dim, dtype=torch.float32, device=q.device)
    check(load().accel_b200_attention(_p(q), _p(k), _p(v), _p(out), seq, position, heads, kv_heads, head_dim, _s()))
    return out


def silu_mul(gate, up):
    check(load().accel_b200_silu_mul(_p(gate), _p(up), gate.numel(), _s()))
    return gate


def residual_add(dest, extra):
    check(load().accel_b200_residual_add(_p(dest), _p(extra), dest.numel(), _s()))
    return dest


def sample(logits, vocab, temperature, rng_state, top_k, chosen=None, index=0):
    chosen = chosen if chosen is not None else torch.full((index + 1,), -1, dtype=torch.int32, device=logits.device)
    check(load().accel_b200_sample(_p(logits), _p(chosen), index, vocab, temperature, _p(rng_state), top_k, _s()))
    return chosen


def argmax_rows(logits):
    rows, vocab = logits.shape
    chosen = torch.full((rows,), -1, dtype=torch.int32, device=logits.device)
    check(load().accel_b200_argmax_rows(_p(logits), rows, vocab, logits.stride(0), _p(chosen), 1, 0, _s()))
    return chosen


def sample_rows(logits, temperature, rng_states, top_k):
    rows, vocab = logits.shape
    chosen = torch.full((rows,), -1, dtype=torch.int32, device=logits.device)
    check(load().accel_b200_sample_rows(_p(logits), rows, vocab, logits.stride(0), _p(chosen), 1, 0, temperature,
                                        _p(rng_states), top_k, _s()))
    return chosen


def matmul_exact(a, b):
    m, k = a.shape
    n = b.shape[1]
    c = torch.full((m, n), 7.0, dtype=torch.float32, device=a.device)
    check(load().accel_b200_matmul(_p(a), _p(b), _p(c), m, k, n, _s()))
    return c


def transpose(src):
    rows, cols = src.shape
    dst = torch.zeros(cols, rows, dtype=torch.float32, device=src.device)
    check(load().accel_b200_transpose(_p(src), _p(dst), rows, cols, _s()))
    return dst


def gemm_epilogue(c, alpha, bias, bias_shape, beta, act):
    m, n = c.shape
    shape = (ctypes.c_int64 * max(1, len(bias_shape)))(*bias_shape)
    check(load().accel_b200_gemm_epilogue(_p(c), m, n, alpha, _p(bias), ctypes.cast(shape, P_i64),
                                          len(bias_shape) if bias is not None else 0, beta, ACT[act], _s()))
    return c


EP_TRIGGER_AFTER_WAIT = 1  # ACCEL_B200_EP_TRIGGER_AFTER_WAIT
ATTN_CACHE_BEFORE_WAIT = 1  # ACCEL_B200_ATTN_CACHE_BEFORE_WAIT


def make_epilogue(alpha=1.0, beta=0.0, bias=None, bias_strides=(0, 0), act="none", residual=None, row_sq=None,
                  flags=0):
    """row_sq: a float64 [m, ceil(n / 128)] tensor that receives each row's
    sums of squares of the outputs per 128-column block. flags: launch
    options (EP_TRIGGER_AFTER_WAIT)."""
    ep = Epilogue()
    ep.alpha, ep.beta = alpha, beta
    ep.bias = 0 if bias is None else bias.data_ptr()
    ep.bias_row_stride, ep.bias_col_stride = bias_strides
    ep.act = ACT[act]
    ep.residual = 0 if residual is None else residual.data_ptr()
    ep.residual_ld = 0 if residual is None else residual.stride(0)
    ep.row_sq = 0 if row_sq is None else row_sq.data_ptr()
    ep.row_sq_ld = 0 if row_sq is None else row_sq.stride(0)
    ep.flags = flags
    # The struct holds raw addresses: keep the tensors alive with it.
    ep._keep = (bias, residual, row_sq)
    return ep


class Workspace:
    """Grows a zero-filled device byte buffer on demand (the kernels keep
    arrival counters in it and leave them zero)."""

    def __init__(self, device="cuda"):
        self.device = device
        self.buf = None

    def get(self, nbytes):
        if nbytes == 0:
            return None
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        return self.buf


def set_q8_path(path):
    """0: by shape (tensor cores where eligible), 1: CUDA cores only."""
    check(load().accel_b200_set_q8_path(path))


_WS = {}


def _workspace(device, nbytes):
    ws = _WS.setdefault(str(device), Workspace(device))
    return ws.get(nbytes)


def matmul_q8(a, q, scale, zero=None, axis=1, epilogue=None, out=None, offset=0, workspace=None):
    """a [m, k] fp32, q int8 holding a [k, n] plane (at `offset`)."""
    lib = load()
    m, k = a.shape
    n = q.shape[-1]
    c = out if out is not None else torch.zeros(m, n, dtype=torch.float32, device=a.device)
    plane = Q8Plane(q.data_ptr(), scale.data_ptr(), 0 if zero is None else zero.data_ptr(), offset, axis)
    need = lib.accel_b200_matmul_q8_workspace(m, k, n)
    ws = workspace if workspace is not None else _workspace(a.device, need)
    check(lib.accel_b200_matmul_q8(_p(a), a.stride(0), ctypes.byref(plane), _p(c), c.stride(0), m, k, n,
                                   None if epilogue is None else ctypes.byref(epilogue), _p(ws),
                                   0 if ws is None else ws.numel(), _s()))
    return c


def matmul_q8_silu(gate_up, q, scale, axis=1, epilogue=None, out=None, workspace=None):
    """SiluMul(gate_up[:, :inter], gate_up[:, inter:]) @ dequant(q); q holds a
    [inter, n] plane."""
    lib = load()
    m, two_inter = gate_up.shape
    inter = two_inter // 2
    n = q.shape[-1]
    c = out if out is not None else torch.zeros(m, n, dtype=torch.float32, device=gate_up.device)
    plane = Q8Plane(q.data_ptr(), scale.data_ptr(), 0, 0, axis)
    need = lib.accel_b200_matmul_q8_silu_workspace(m, inter, n)
    ws = workspace if workspace is not None else _workspace(gate_up.device, need)
    check(lib.accel_b200_matmul_q8_silu(_p(gate_up), gate_up.stride(0), inter, ctypes.byref(plane), _p(c), c.stride(0),
                                        m, n, None if epilogue is None else ctypes.byref(epilogue), _p(ws),
                                        0 if ws is None else ws.numel(), _s()))
    return c


def matmul_q8_rmsnorm(x, gamma, eps, q, scale, axis=1, epilogue=None, out=None, workspace=None):
    """RmsNorm(x[:, :k]) @ dequant(q); q holds a [k, n] plane (x's row stride
    may be wider than k)."""
    lib = load()
    m = x.shape[0]
    k, n = q.shape
    c = out if out is not None else torch.zeros(m, n, dtype=torch.float32, device=x.device)
    plane = Q8Plane(q.data_ptr(), scale.data_ptr(), 0, 0, axis)
    need = lib.accel_b200_matmul_q8_rmsnorm_workspace(m, k, n)
    ws = workspace if workspace is not None else _workspace(x.device, need)
    check(lib.accel_b200_matmul_q8_rmsnorm(_p(x), x.stride(0), _p(gamma), eps, ctypes.byref(plane), _p(c), c.stride(0),
                                           m, k, n, None if epilogue is None else ctypes.byref(epilogue), _p(ws),
                                           0 if ws is None else ws.numel(), _s()))
    return c


def matmul_q8_rmsnorm_stats(x, row_sq, gamma, eps, q, scale, axis=1, epilogue=None, out=None, workspace=None):
    """RmsNorm(x[:, :k]) @ dequant(q) with each row's sum of squares given as
    row_sq [m, blocks] (float64 partial sums, added in order)."""
    lib = load()
    m = x.shape[0]
    k, n = q.shape
    c = out if out is not None else torch.zeros(m, n, dtype=torch.float32, device=x.device)
    plane = Q8Plane(q.data_ptr(), scale.data_ptr(), 0, 0, axis)
    need = lib.accel_b200_matmul_q8_rmsnorm_workspace(m, k, n)
    ws = workspace if workspace is not None else _workspace(x.device, need)
    check(lib.accel_b200_matmul_q8_rmsnorm_stats(_p(x), x.stride(0), _p(row_sq), row_sq.stride(0), row_sq.shape[1],
                                                 _p(gamma), eps, ctypes.byref(plane), _p(c), c.stride(0), m, k, n,
                                                 None if epilogue is None else ctypes.byref(epilogue), _p(ws),
                                                 0 if ws is None else ws.numel(), _s()))
    return c


def pair_gate_up(gate_up, inter):
    """Columns [gate (inter) | up (inter)] of a weight (or a scale vector) in
    the 64-column pairs accel_b200_matmul_q8_rmsnorm_silu_pairs reads: block
    t holds gate columns 64t .. 64t + 63, then the same up columns."""
    lead = gate_up.shape[:-1]
    g = gate_up[..., :inter].reshape(*lead, inter // 64, 64)
    u = gate_up[..., inter:].reshape(*lead, inter // 64, 64)
    return torch.stack([g, u], dim=-2).reshape(*lead, 2 * inter).contiguous()


def matmul_q8_rmsnorm_silu_pairs(x, gamma, eps, q, scale, row_sq=None, axis=1, out=None, workspace=None):
    """SiluMul(gate, up) of RmsNorm(x[:, :k]) @ dequant(q), q's columns in
    64-column gate|up pairs (pair_gate_up); the result has n / 2 columns.
    row_sq: optional [m, blocks] float64 sums of squares of x's rows."""
    lib = load()
    m = x.shape[0]
    k, n = q.shape
    c = out if out is not None else torch.zeros(m, n // 2, dtype=torch.float32, device=x.device)
    plane = Q8Plane(q.data_ptr(), scale.data_ptr(), 0, 0, axis)
    need = lib.accel_b200_matmul_q8_rmsnorm_workspace(m, k, n)
    ws = workspace if workspace is not None else _workspace(x.device, need)
    sq_ld, sq_n = (row_sq.stride(0), row_sq.shape[1]) if row_sq is not None else (0, 0)
    check(lib.accel_b200_matmul_q8_rmsnorm_silu_pairs(_p(x), x.stride(0), _p(row_sq), sq_ld, sq_n, _p(gamma), eps,
                                                      ctypes.byref(plane), _p(c), c.stride(0), m, k, n, _p(ws),
                                                      0 if ws is None else ws.numel(), _s()))
    return c


def matmul_f32(a, b, epilogue=None, out=None):
    lib = load()
    m, k = a.shape
    n = b.shape[1]
    c = out if out is not None else torch.zeros(m, n, dtype=torch.float32, device=a.device)
    need = lib.accel_b200_matmul_f32_workspace(m, k, n)
    ws = _workspace(a.device, need)
    check(lib.accel_b200_matmul_f32(_p(a), a.stride(0), _p(b), _p(c), c.stride(0), m, k, n,
                                    None if epilogue is None else ctypes.byref(epilogue), _p(ws),
                                    0 if ws is None else ws.numel(), _s()))
    return c


def attention_decode(q, k_cache, v_cache, lens, heads, kv_heads, head_dim, max_len, chunk=64, head_major=False,
                     workspace=None, status=None):
    """q [B, heads * head_dim]. Caches [B, max_len, kv_heads, head_dim] (the
    reference layout) or, with head_major, [B, kv_heads, max_len, head_dim]."""
    lib = load()
    batch = q.shape[0]
    out = torch.zeros(batch, heads * head_dim, dtype=torch.float32, device=q.device)
    need = lib.accel_b200_attention_decode_workspace(batch, heads, kv_heads, max_len, chunk)
    ws = workspace if workspace is not None else torch.zeros(need, dtype=torch.uint8, device=q.device)
    if head_major:
        row, head, seq = head_dim, max_len * head_dim, kv_heads * max_len * head_dim
    else:
        row, head, seq = kv_heads * head_dim, head_dim, max_len * kv_heads * head_dim
    check(lib.accel_b200_attention_decode(_p(q), q.stride(0), _p(k_cache), _p(v_cache), row, head, seq, _p(lens), batch,
                                          heads, kv_heads, head_dim, max_len, chunk, _p(out), out.stride(0), _p(ws),
                                          ws.numel(), _p(status), _s()))
    return out


def rope_append(qkv, row_seq, row_pos, heads, kv_heads, head_dim, cos_t, sin_t, k_cache, v_cache):
    """Rope + AppendCache over fused q|k|v rows (queries rotated in place).
    Caches head-major [slots, kv_heads, context, head_dim]."""
    ctx = k_cache.shape[2]
    check(load().accel_b200_rope_append(_p(qkv), qkv.stride(0), _p(row_seq), _p(row_pos), qkv.shape[0], heads,
                                        kv_heads, head_dim, _p(cos_t), _p(sin_t), _p(k_cache), _p(v_cache),
                                        kv_heads * ctx * head_dim, ctx * head_dim, head_dim, _s()))


def _l2_prefetch(tensors, flags):
    pf = L2Prefetch()
    for i, t in enumerate(tensors):
        pf.ptr[i] = t.data_ptr()
        pf.bytes[i] = t.numel() * t.element_size()
    pf.count = len(tensors)
    pf.flags = flags
    return pf


def decode_attention(qkv, row_pos, heads, kv_heads, cos_t, sin_t, k_cache, v_cache, row_seq=None, out=None,
                     status=None, prefetch=None, flags=0):
    """Fused decode step (Rope, AppendCache, attention) over un-rotated q|k|v
    rows; caches head-major [slots, kv_heads, context, 64]. prefetch: up to
    four contiguous device tensors to bring into L2 meanwhile (a hint).
    flags: launch options (ATTN_CACHE_BEFORE_WAIT)."""
    rows, ctx = qkv.shape[0], k_cache.shape[2]
    if out is None:
        out = torch.zeros(rows, heads * 64, dtype=torch.float32, device=qkv.device)
    args = (_p(qkv), qkv.stride(0), _p(row_seq), _p(row_pos), rows, heads, kv_heads, 64, _p(cos_t), _p(sin_t), ctx,
            _p(k_cache), _p(v_cache), kv_heads * ctx * 64, ctx * 64, _p(out), out.stride(0), _p(status))
    if prefetch is None and flags == 0:
        check(load().accel_b200_decode_attention(*args, _s()))
    else:
        pf = _l2_prefetch(prefetch or [], flags)
        check(load().accel_b200_decode_attention_prefetch(*args, ctypes.byref(pf), _s()))
    return out


def attention_prefill(q, k_cache, v_cache, first, count, pos0, heads, kv_heads, out=None, max_rows=None):
    """Tiled causal prefill attention. q [rows, heads * 64] (roped); caches
    head-major [slots, kv_heads, context, 64]; first/count/pos0 int32 [batch]
    device tensors."""
    rows = q.shape[0]
    ctx = k_cache.shape[2]
    if out is None:
        out = torch.zeros(rows, heads * 64, dtype=torch.float32, device=q.device)
    batch = first.shape[0]
    if max_rows is None:
        max_rows = int(count.max().item()) if batch else 0
    check(load().accel_b200_attention_prefill(_p(q), q.stride(0), _p(k_cache), _p(v_cache), kv_heads * ctx * 64,
                                              ctx * 64, _p(out), out.stride(0), _p(first), _p(count), _p(pos0), batch,
                                              max_rows, heads, kv_heads, 64, _s()))
    return out


def attention_decode_workspace(batch, heads, kv_heads, max_len, chunk=64, device="cuda"):
    """A zeroed workspace for attention_decode (its counters start at zero)."""
    need = load().accel_b200_attention_decode_workspace(batch, heads, kv_heads, max_len, chunk)
    return torch.zeros(need, dtype=torch.uint8, device=device)


class Q8Cache:
    """An int8 key/value cache (accel_b200_q8_cache) over torch tensors: k and
    v int8 [slots, kv_heads, context, head_dim] and their fp32 scales [slots,
    kv_heads, ceil(context / block)], all on one CUDA device. The planes may be
    views of larger ones as long as a (slot, head) run is contiguous."""

    def __init__(self, k, v, k_scale, v_scale, block=64):
        slots, kv_heads, context, head_dim = k.shape
        if block not in (32, 64, 128):
            raise ValueError("block must be 32, 64 or 128 tokens")
        blocks = -(-context // block)
        for name, t, dtype, shape in (("k", k, torch.int8, k.shape), ("v", v, torch.int8, k.shape),
                                      ("k_scale", k_scale, torch.float32, (slots, kv_heads, blocks)),
                                      ("v_scale", v_scale, torch.float32, (slots, kv_heads, blocks))):
            if t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != k.device or not t.is_cuda:
                raise ValueError(f"{name} must be {dtype} {tuple(shape)} on one CUDA device")
        if k.stride() != v.stride() or k_scale.stride() != v_scale.stride():
            raise ValueError("k and v (and their scales) must have the same strides")
        if k.stride(3) != 1 or (k.stride(2) != head_dim and context > 1) or (k_scale.stride(2) != 1 and blocks > 1):
            raise ValueError("a (slot, head) run of the cache must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale, self.block = k, v, k_scale, v_scale, block
        self.slots, self.kv_heads, self.context, self.head_dim = slots, kv_heads, context, head_dim
        self.device, self.index = k.device, k.get_device()
        self.native = Q8CacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.stride(0),
                                    k.stride(1), k_scale.stride(0), k_scale.stride(1), slots, kv_heads, head_dim,
                                    context, block)
        self._ref = ctypes.byref(self.native)

    @classmethod
    def zeros(cls, slots, kv_heads, context, head_dim, block=64, device="cuda"):
        if block not in (32, 64, 128):
            raise ValueError("block must be 32, 64 or 128 tokens")
        planes = [torch.zeros(slots, kv_heads, context, head_dim, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(slots, kv_heads, -(-context // block), device=device) for _ in range(2)]
        return cls(*planes, *scales, block)


_FLOAT32, _INT32 = torch.float32, torch.int32


def _rows(name, t, index, width):
    """(rows, row stride) of a 2-D fp32 tensor of `width` columns on device `index`."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not _FLOAT32 or t.get_device() != index or len(shape) != 2 or shape[1] != width or stride[1] != 1:
        raise ValueError(f"{name} must be fp32 [rows, {width}] with contiguous rows on cuda:{index}")
    rows = shape[0]
    # One row has no stride that matters (torch reports that of the tensor it was cut from).
    return rows, stride[0] if rows > 1 else width


def _i32(name, t, index, n):
    """The address of n contiguous int32 on device `index` (None: 0)."""
    if t is None:
        return 0
    if t.numel() == n and t.dtype is _INT32 and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name} must be {n} contiguous int32 on cuda:{index}")


def _counts(bits):
    """Refuses numbers (or-ed together) that a C int would hold as others."""
    if bits >> 31:
        raise ValueError("rows, windows and sinks are counts of 31 bits")


def _table(name, t, cache):
    shape = t.shape
    if (t.dtype is not torch.float32 or t.get_device() != cache.index or len(shape) != 2 or
            shape[0] < cache.context or shape[1] != cache.head_dim or not t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous fp32 [context, head_dim] on cuda:{cache.index}")
    return t.data_ptr()


def _bytes(ws, index):
    """(address, size) of a workspace on device `index` (None: none)."""
    if ws is None:
        return 0, 0
    if ws.dtype is not torch.uint8 or ws.get_device() != index or not ws.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on cuda:{index}")
    return ws.data_ptr(), ws.numel()


def _call(index, fn, *args):
    """fn(*args, stream) with device `index` current, on its current stream. (A
    decode step makes these calls once per layer: the raw stream and device
    numbers spare the objects that torch's public calls build.)"""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        check(fn(*args, stream))
    else:
        with torch.cuda.device(index):
            check(fn(*args, stream))


def rope_append_q8(qkv, cache, first, count, pos0, heads, max_rows, cos_t, sin_t, q_out=None, status=None):
    """Rope and quantising append: sequence b's rows first[b] .. + count[b] - 1
    of qkv [rows, (heads + 2 kv_heads) * head_dim] at positions pos0[b] + i of
    slot b (int32 device vectors; count[b] <= max_rows). Returns the roped
    queries [rows, heads * head_dim] (q_out; rows of no sequence are left)."""
    index, d = cache.index, cache.head_dim
    rows, ld = _rows("qkv", qkv, index, (heads + 2 * cache.kv_heads) * d)
    batch = first.numel()
    if q_out is None:
        q_out = torch.zeros(rows, heads * d, dtype=torch.float32, device=cache.device)
    q_rows, q_ld = _rows("q_out", q_out, index, heads * d)
    if q_rows != rows:
        raise ValueError("q_out must have a row for each row of qkv")
    _counts(max_rows)
    if rows == 0 or batch == 0:
        return q_out
    _call(index, load().accel_b200_rope_append_q8, qkv.data_ptr(), ld, rows, cache._ref,
          _i32("first", first, index, batch), _i32("count", count, index, batch), _i32("pos0", pos0, index, batch),
          batch, max_rows, heads, _table("cos_t", cos_t, cache), _table("sin_t", sin_t, cache), q_out.data_ptr(), q_ld,
          _i32("status", status, index, 1))
    return q_out


def cache_rows_q8(cache, first, count, pos0, max_rows, k_out=None, v_out=None, status=None):
    """Cache positions pos0[b] + i of slot b as fp32 into rows first[b] + i of
    k_out and v_out [rows, kv_heads * head_dim] (either may be None)."""
    index, width, batch = cache.index, cache.kv_heads * cache.head_dim, first.numel()
    k = v = None
    if k_out is not None:
        k = _rows("k_out", k_out, index, width)
    if v_out is not None:
        v = _rows("v_out", v_out, index, width)
    if (k or v) is None or (k is not None and v is not None and k != v):
        raise ValueError("k_out and v_out must have the same rows and strides, and one must be given")
    rows, ld = k or v
    _counts(max_rows)
    if rows == 0 or batch == 0:
        return k_out, v_out
    _call(index, load().accel_b200_cache_rows_q8, cache._ref, _i32("first", first, index, batch),
          _i32("count", count, index, batch), _i32("pos0", pos0, index, batch), batch, max_rows,
          0 if k is None else k_out.data_ptr(), 0 if v is None else v_out.data_ptr(), ld, rows,
          _i32("status", status, index, 1))
    return k_out, v_out


def _attention_io(q, cache, heads, out):
    """(rows, q's row stride, out, out's row stride)."""
    width = heads * cache.head_dim
    rows, q_ld = _rows("q", q, cache.index, width)
    if out is None:
        out = torch.zeros(rows, width, dtype=torch.float32, device=cache.device)
    out_rows, out_ld = _rows("out", out, cache.index, width)
    if out_rows != rows:
        raise ValueError("out must have a row for each row of q")
    return rows, q_ld, out, out_ld


def attention_decode_q8_workspace(cache, rows, heads, window=0, sinks=0):
    """A zeroed workspace for attention_decode_q8 calls of these sizes (None:
    none needed)."""
    _counts(rows | window | sinks)
    need = load().accel_b200_attention_decode_q8_workspace(cache._ref, rows, heads, window, sinks)
    return torch.zeros(need, dtype=torch.uint8, device=cache.device) if need else None


def attention_decode_q8(q, cache, row_pos, heads, row_seq=None, window=0, sinks=0, out=None, workspace=None,
                        status=None, prefetch=None, flags=0):
    """Attention of roped query rows q [rows, heads * head_dim], row r at
    position row_pos[r] of slot row_seq[r] (None: slot r), over an int8 cache.
    window: how many of the last tokens a row sees (0: all); sinks: first
    tokens it sees besides. Rows with row_pos < 0 are left. prefetch: up to
    four contiguous device tensors to bring into L2 meanwhile; flags: launch
    options (ATTN_CACHE_BEFORE_WAIT)."""
    index = cache.index
    rows, q_ld, out, out_ld = _attention_io(q, cache, heads, out)
    _counts(window | sinks)
    if rows == 0:
        return out
    if workspace is None:
        workspace = attention_decode_q8_workspace(cache, rows, heads, window, sinks)
    ws, ws_bytes = _bytes(workspace, index)
    args = (q.data_ptr(), q_ld, cache._ref, _i32("row_seq", row_seq, index, rows),
            _i32("row_pos", row_pos, index, rows), rows, heads, window, sinks, out.data_ptr(), out_ld, ws, ws_bytes,
            _i32("status", status, index, 1))
    if prefetch is None and flags == 0:
        _call(index, load().accel_b200_attention_decode_q8, *args)
    else:
        for t in prefetch or []:
            if t.get_device() != index or not t.is_contiguous():
                raise ValueError(f"prefetch takes contiguous tensors on cuda:{index}")
        _call(index, load().accel_b200_attention_decode_q8_prefetch, *args,
              ctypes.byref(_l2_prefetch(prefetch or [], flags)))
    return out


def attention_prefill_q8_workspace(cache, batch, max_rows, heads, window=0, sinks=0):
    """A zeroed workspace for attention_prefill_q8 calls of these sizes (None:
    none needed)."""
    _counts(batch | max_rows | window | sinks)
    need = load().accel_b200_attention_prefill_q8_workspace(cache._ref, batch, max_rows, heads, window, sinks)
    return torch.zeros(need, dtype=torch.uint8, device=cache.device) if need else None


def attention_prefill_q8_tiles(cache, batch, max_rows, heads, window=0, sinks=0):
    """Whether attention_prefill_q8 calls of these sizes take the tcgen05 tiles
    (else the groups of 8 query vectors)."""
    _counts(batch | max_rows | window | sinks)
    return bool(load().accel_b200_attention_prefill_q8_tiles(cache._ref, batch, max_rows, heads, window, sinks))


def attention_prefill_q8(q, cache, first, count, pos0, heads, max_rows, window=0, sinks=0, out=None, workspace=None,
                         status=None):
    """Causal attention of sequence b's rows first[b] .. + count[b] - 1 of q
    (roped) at positions pos0[b] + i over slot b of an int8 cache that holds
    their keys and values. window and sinks as in attention_decode_q8."""
    index, batch = cache.index, first.numel()
    rows, q_ld, out, out_ld = _attention_io(q, cache, heads, out)
    _counts(max_rows | window | sinks)
    if rows == 0 or batch == 0:
        return out
    if workspace is None:
        workspace = attention_prefill_q8_workspace(cache, batch, max_rows, heads, window, sinks)
    ws, ws_bytes = _bytes(workspace, index)
    _call(index, load().accel_b200_attention_prefill_q8, q.data_ptr(), q_ld, cache._ref,
          _i32("first", first, index, batch), _i32("count", count, index, batch), _i32("pos0", pos0, index, batch),
          batch, max_rows, rows, heads, window, sinks, out.data_ptr(), out_ld, ws, ws_bytes,
          _i32("status", status, index, 1))
    return out
