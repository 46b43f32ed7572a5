"""Torch-facing wrappers of the gfx950 kernels (device tensors in, device tensors out).

Each op checks dtypes, devices and contiguity, allocates its outputs with PyTorch's caching
allocator on the input's device, launches on that device's current stream and raises
``RuntimeError`` (with the library's message) on any failure.  No op has a CPU implementation:
on a tensor that is not on a GPU they raise ``RuntimeError``.
"""
import contextlib
import ctypes
import threading

import torch

from . import _native

# Opt-in launch timing: while kernel_timer() is active, every launch is bracketed by a pair of
# HIP events recorded on the stream it runs on (the device's current stream).
_timer = None


@contextlib.contextmanager
def kernel_timer():
    """Collect {op name: [(start event, end event), ...]} for the launches inside the block."""
    global _timer
    prev, _timer = _timer, {}
    try:
        yield _timer
    finally:
        _timer = prev


def kernel_times_ms(events):
    """{op: [milliseconds per launch]} from kernel_timer()'s events (synchronizes)."""
    torch.cuda.synchronize()
    return {k: [a.elapsed_time(b) for a, b in v] for k, v in events.items()}


def _launch(name, fn, *args):
    if _timer is None:
        return _native.check(fn(*args), name)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    status = fn(*args)
    b.record()
    _timer.setdefault(name, []).append((a, b))
    return _native.check(status, name)

_DT = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32}


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


try:   # the current stream's raw handle without building a torch.cuda.Stream (2.4 -> ~0.3 us a call)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    _raw_stream = None


def _stream(t):
    if _raw_stream is not None:
        return ctypes.c_void_p(_raw_stream(t.device.index))
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _raw(index):
    """The current stream of device `index` as an integer."""
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _call(name, fn, *args):
    """_launch for integer arguments."""
    if _timer is not None:
        return _launch(name, fn, *args)
    status = fn(*args)
    if status:
        _native.check(status, name)


def _need_gpu(*tensors):
    for t in tensors:
        if t is not None and t.device.type != "cuda":
            raise RuntimeError(f"psquant kernels need GPU tensors (got {t.device})")


def _dt(t, what):
    if t.dtype not in _DT:
        raise TypeError(f"{what}: unsupported dtype {t.dtype}")
    return _DT[t.dtype]


def _rows2d(x):
    """[M, K] with unit column stride, rows at least K apart and 16-byte aligned rows: x itself
    when it is so laid out, else a packed copy (torch's contiguous() keeps the strides of size-1
    dimensions and the offset of an aligned-looking view, so the copy is explicit)."""
    if x.dim() != 2:
        raise ValueError("expected a 2-D tensor")
    M, K = x.shape
    if M == 0 or K == 0:
        return x
    if (x.stride(1) != 1 or x.stride(0) < K or (x.stride(0) * x.element_size()) % 16
            or x.data_ptr() % 16):
        x = torch.empty((M, K), dtype=x.dtype, device=x.device).copy_(x)
    return x


def _bias(bias, n, device):
    if bias is None:
        return None, 0
    if bias.numel() != n:
        raise ValueError(f"bias has {bias.numel()} elements, expected {n}")
    bias = bias.to(device).contiguous()
    return bias, _dt(bias, "bias")


# ------------------------------------------------------------------ activations
def quantize_rows(x, fp8=False, rot_group=0, static_scale=None):
    """Fused ConvRot rotation + per-row absmax + int8 (or fp8 e4m3fn) quantization.

    x: [M, K] bf16/f16 on the GPU.  Returns (q [M, K] int8 or float8_e4m3fn, scale [M] fp32).
    static_scale: optional fp32 tensor with one element (the module's input_scale).
    """
    _need_gpu(x, static_scale)
    x = _rows2d(x)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"quantize_rows: activations must be bf16/f16, got {x.dtype}")
    M, K = x.shape
    q = torch.empty(M, K, dtype=torch.float8_e4m3fn if fp8 else torch.int8, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    st = None
    if static_scale is not None:
        st = static_scale.to(device=x.device, dtype=torch.float32).reshape(-1)[:1].contiguous()
    fn = _native.lib().psq_quantize_rows_fp8 if fp8 else _native.lib().psq_quantize_rows_i8
    _launch("quantize_rows_fp8" if fp8 else "quantize_rows_i8", fn, _p(x), _DT[x.dtype], M, K, x.stride(0),
            int(rot_group or 0), _p(st), _p(q), K, _p(scale), _stream(x))
    return q, scale


def rotate_rows(x, rot_group, out_dtype=None):
    """x H per group of rot_group elements (the quantizer's fixed-order transform, one rounding to
    out_dtype, default x.dtype).  x: [M, K] bf16/f16 on the GPU; rot_group 0 converts only."""
    _need_gpu(x)
    x = _rows2d(x)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"rotate_rows: activations must be bf16/f16, got {x.dtype}")
    M, K = x.shape
    y = torch.empty(M, K, dtype=out_dtype or x.dtype, device=x.device)
    _launch("rotate_rows", _native.lib().psq_rotate_rows, _p(x), _DT[x.dtype], M, K, x.stride(0), int(rot_group or 0),
            _p(y), _dt(y, "out"), K, _stream(x))
    return y


# ----------------------------------------------------------------------- GEMMs
# epilogue activations of the W8A8 / FP8 GEMMs (enum psq_activation)
ACTIVATIONS = {None: 0, "none": 0, "gelu_tanh": 1, "silu_gate": 2}


def _act(activation):
    try:
        return ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"unknown epilogue activation {activation!r}") from None


def _out_cols(N, act, name):
    """Output columns: N, or N / 2 for the SiLU gate (gate rows, then up rows)."""
    if act != ACTIVATIONS["silu_gate"]:
        return N
    if N % 128:
        raise ValueError(f"{name}: the SiLU gate needs N (gate + up rows) a multiple of 128, got {N}")
    return N // 2


def gemm_i8(a, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, activation=None):
    """y = round(fmaf(a @ w.T (int32), a_scale[m] * w_scale[n], bias[n])): [M, N] out_dtype.

    activation "gelu_tanh": y = round(gelu_tanh(round(...))) -- the GELU of the rounded output,
    rounded again (the Wan FFN's F.gelu(fc1(x).float(), approximate="tanh") then fc2's cast).
    activation "silu_gate": w holds N / 2 gate rows then N / 2 up rows (N a multiple of 128);
    y[m, j] = round(silu(round(g)) * round(u)) is [M, N / 2], g and u the linear outputs of
    columns j and N / 2 + j (the H3 MLP's F.silu(gate.float()) * up.float(), then fc2's cast).
    """
    _need_gpu(a, a_scale, w, w_scale)
    a, w = _rows2d(a), _rows2d(w)
    if a.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError("gemm_i8: operands must be int8")
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"gemm_i8: K mismatch {K} vs {w.shape[1]}")
    a_scale = a_scale.to(torch.float32).reshape(-1).contiguous()
    w_scale = w_scale.to(torch.float32).reshape(-1).contiguous()
    if a_scale.numel() != M or w_scale.numel() != N:
        raise ValueError("gemm_i8: scale sizes do not match M / N")
    bias, bdt = _bias(bias, N, a.device)
    act = _act(activation)
    y = torch.empty(M, _out_cols(N, act, "gemm_i8"), dtype=out_dtype, device=a.device)
    if act:
        _launch("gemm_i8", _native.lib().psq_gemm_i8_act, _p(a), a.stride(0), _p(a_scale), _p(w), w.stride(0), _p(w_scale),
                _p(bias), bdt, act, _p(y), _dt(y, "out"), y.shape[1], M, N, K, _stream(a))
    else:
        _launch("gemm_i8", _native.lib().psq_gemm_i8, _p(a), a.stride(0), _p(a_scale), _p(w), w.stride(0), _p(w_scale),
                _p(bias), bdt, _p(y), _dt(y, "out"), N, M, N, K, _stream(a))
    return y


def gemm_i8_i32(a, w):
    """Raw int32 accumulators a @ w.T ([M, N] int32)."""
    _need_gpu(a, w)
    a, w = _rows2d(a), _rows2d(w)
    M, K = a.shape
    N = w.shape[0]
    c = torch.empty(M, N, dtype=torch.int32, device=a.device)
    _launch("gemm_i8_i32", _native.lib().psq_gemm_i8_i32, _p(a), a.stride(0), _p(w), w.stride(0), _p(c), N, M, N, K, _stream(a))
    return c


def gemm_fp8(a, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, activation=None):
    """fp8 GEMM: y = round(fmaf(a @ w.T (fp32), a_scale[m] * w_scale[n or 0], bias[n])).

    a: e4m3fn activation codes.  w: e4m3fn codes, or float8_e5m2 codes (``psq_gemm_fp8_e5m2w``,
    no activation epilogue).  uint8 views are read as e4m3fn.  activation as in gemm_i8.
    """
    _need_gpu(a, a_scale, w, w_scale)
    a, w = _rows2d(a), _rows2d(w)
    if a.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError("gemm_fp8: activations must be float8_e4m3fn")
    e5m2 = w.dtype == torch.float8_e5m2
    if w.dtype not in (torch.float8_e4m3fn, torch.uint8) and not e5m2:
        raise TypeError("gemm_fp8: weights must be float8_e4m3fn or float8_e5m2")
    if e5m2 and activation not in (None, "none"):
        raise ValueError("gemm_fp8: float8_e5m2 weights take no activation epilogue")
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"gemm_fp8: K mismatch {K} vs {w.shape[1]}")
    a_scale = a_scale.to(torch.float32).reshape(-1).contiguous()
    w_scale = w_scale.to(device=a.device, dtype=torch.float32).reshape(-1).contiguous()
    if a_scale.numel() != M or w_scale.numel() not in (1, N):
        raise ValueError("gemm_fp8: scale sizes do not match")
    bias, bdt = _bias(bias, N, a.device)
    act = _act(activation)
    y = torch.empty(M, _out_cols(N, act, "gemm_fp8"), dtype=out_dtype, device=a.device)
    if act:
        _launch("gemm_fp8", _native.lib().psq_gemm_fp8_act, _p(a), a.stride(0), _p(a_scale), _p(w), w.stride(0),
                _p(w_scale), int(w_scale.numel() > 1), _p(bias), bdt, act, _p(y), _dt(y, "out"), y.shape[1], M, N, K,
                _stream(a))
    else:
        fn = _native.lib().psq_gemm_fp8_e5m2w if e5m2 else _native.lib().psq_gemm_fp8
        _launch("gemm_fp8", fn, _p(a), a.stride(0), _p(a_scale), _p(w), w.stride(0),
                _p(w_scale), int(w_scale.numel() > 1), _p(bias), bdt, _p(y), _dt(y, "out"), N, M, N, K, _stream(a))
    return y


# Workspaces of the weight-only GEMMs (split K) and of paged_attention (split length), one per (device,
# stream): launches on one stream run in order, so calls of one launch can share it, whichever host thread makes
# them (calls on two streams would race on its counters).  A call of two launches, between which another thread's
# could come, has memory of its own (paged_attention whose parts a second kernel joins).  A call that needs
# more gets a larger one (at least twice the size, so a stream is replaced a few times at most), and
# the replaced buffer is kept until the process ends: a launch captured into a graph keeps the
# address it was given, which must not be handed out again.  None is made or replaced during a capture: a
# captured call without one that is large enough runs unsplit.  Replays of a graph use the workspace of the stream
# that captured it, so they must not overlap with each other or with that stream's calls.  At most _MAX_WS_STREAMS streams per
# device get one; calls on further streams run without a workspace (the data-parallel tiles: the
# same results, the split of K left out).  For capture and for callers that cannot allocate at all,
# psq_gemm_w4a16_noalloc uses the library's own static scratch instead.
_workspaces = {}
_retired_workspaces = []
_workspaces_lock = threading.Lock()
_MAX_WS_STREAMS = 16
_WS_MIN_BYTES = 1 << 20


def _workspace(device, stream, nbytes):
    if nbytes <= 0:
        return None, 0
    key = (device.index, stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        with _workspaces_lock:
            ws = _larger_workspace(key, device, nbytes)
        if ws is None:
            return None, 0
    return ws, ws.numel()


def _larger_workspace(key, device, nbytes):
    ws = _workspaces.get(key)
    if ws is not None and ws.numel() >= nbytes:   # another thread was first
        return ws
    if ws is None and sum(1 for d, _ in _workspaces if d == device.index) >= _MAX_WS_STREAMS:
        return None
    if torch.cuda.is_current_stream_capturing():
        return None   # (the zeros would be the graph's: later calls would find counters that only its replays zero)
    size = max(nbytes, _WS_MIN_BYTES, 2 * ws.numel() if ws is not None else 0)
    if ws is not None:
        _retired_workspaces.append(ws)
    ws = torch.zeros(size, dtype=torch.uint8, device=device)   # counter words zero once; calls leave them so
    _workspaces[key] = ws
    return ws


def gemm_w4a16(x, wq, w_scale, w_zero, group_size, bias=None, out_dtype=None):
    """uint4 asymmetric group weights, in-register dequantized onto bf16/f16 MFMA.

    x [M, K] bf16/f16, wq [N, K/2] uint8 (low nibble = even k), w_scale/w_zero [N, K/group] fp16.
    Shapes that leave CUs idle split K across workgroups through a cached workspace.
    """
    _need_gpu(x, wq, w_scale, w_zero)
    x, wq = _rows2d(x), wq.contiguous()
    M, K = x.shape
    N = wq.shape[0]
    if wq.shape[1] * 2 != K:
        raise ValueError(f"gemm_w4a16: packed weight [{N}, {wq.shape[1]}] does not match K={K}")
    w_scale = w_scale.to(torch.float16).contiguous()
    w_zero = w_zero.to(torch.float16).contiguous()
    bias, bdt = _bias(bias, N, x.device)
    y = torch.empty(M, N, dtype=out_dtype or x.dtype, device=x.device)
    stream = _stream(x)
    ws, nb = _workspace(x.device, stream.value,
                        _native.lib().psq_gemm_wonly_workspace_bytes(_native.W_UINT4, x.stride(0), M, N, K,
                                                                     int(group_size)))
    _launch("gemm_w4a16", _native.lib().psq_gemm_w4a16_ws, _p(x), _dt(x, "x"), x.stride(0), _p(wq), _p(w_scale),
            _p(w_zero), int(group_size), _p(bias), bdt, _p(y), _dt(y, "out"), N, M, N, K, _p(ws), nb, stream)
    return y


def gemm_w8a16(x, wq, w_scale, bias=None, out_dtype=None):
    """int8 weight-only: y = round(fmaf(x @ q.T (fp32), w_scale[n], bias[n]))."""
    _need_gpu(x, wq, w_scale)
    x, wq = _rows2d(x), _rows2d(wq)
    M, K = x.shape
    N = wq.shape[0]
    w_scale = w_scale.to(torch.float32).reshape(-1).contiguous()
    bias, bdt = _bias(bias, N, x.device)
    y = torch.empty(M, N, dtype=out_dtype or x.dtype, device=x.device)
    stream = _stream(x)
    ws, nb = _workspace(x.device, stream.value,
                        _native.lib().psq_gemm_wonly_workspace_bytes(_native.W_INT8, x.stride(0), M, N, K, 0))
    _launch("gemm_w8a16", _native.lib().psq_gemm_w8a16_ws, _p(x), _dt(x, "x"), x.stride(0), _p(wq), _p(w_scale),
            _p(bias), bdt, _p(y), _dt(y, "out"), N, M, N, K, _p(ws), nb, stream)
    return y


# ------------------------------------------------------- module forward in one call
# The launches of a QuantLinear forward with nothing to convert: addresses and sizes straight to the
# library, at most one scratch allocation, no tensor per stored component.  For the small calls, which
# the host bounds: an int8 or fp8 forward 39 -> 17.8 us of host time (one or two rows, quantized inside
# the GEMM: 13.8 us), int4 28 -> 13.5 us.  The arguments are as the general ops check them
# (QuantLinear._direct); None when the library refuses, and the caller's general path then reports why.
def quantized_in_gemm(M, K, act):
    """Whether linear_q8_direct quantizes the rows inside its GEMM (no codes, no scratch: psq_linear_q8)."""
    return M <= 2 and K <= 8192 and act != ACTIVATIONS["silu_gate"]


def linear_q8_direct(x, M, K, weights, w, w_scale, per_row, rot_group, N, bias, act, into=None):
    """x [..., K] contiguous bf16/f16; w, w_scale: device addresses.  [..., N] (gate: N / 2) of x's
    dtype; into: [M, N] rows of x's dtype or fp32 (the same values) that take the result."""
    lib, dt = _native.lib(), _DT[x.dtype]
    cols = _out_cols(N, act, "linear_q8")
    y = torch.empty(x.shape[:-1] + (cols,), dtype=x.dtype, device=x.device) if into is None else into
    scratch = None if M <= 2 and quantized_in_gemm(M, K, act) else \
        torch.empty(((M * K + 15) & -16) + 4 * M, dtype=torch.uint8, device=x.device)
    status = lib.psq_linear_q8(weights, x.data_ptr(), dt, K, rot_group, w, K, w_scale, per_row,
                               None if bias is None else bias.data_ptr(), dt, act, y.data_ptr(),
                               int(y.dtype is torch.float32), cols, M, N, K,
                               None if scratch is None else scratch.data_ptr(),
                               _raw_stream(x.device.index))
    return None if status else y


def quantize_direct(x, M, K, fp8, rot_group):
    """quantize_rows of x [..., K] contiguous bf16/f16: (codes [M, K], scales [M])."""
    lib = _native.lib()
    q = torch.empty(M, K, dtype=torch.float8_e4m3fn if fp8 else torch.int8, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    status = (lib.psq_quantize_rows_fp8 if fp8 else lib.psq_quantize_rows_i8)(
        x.data_ptr(), _DT[x.dtype], M, K, K, rot_group, None, q.data_ptr(), K, scale.data_ptr(), _raw_stream(x.device.index))
    return None if status else (q, scale)


def linear_codes_direct(x, q, scale, M, K, weights, w, w_scale, per_row, N, bias, act):
    """linear_q8_direct of rows that are quantized already (q, scale: quantize_direct of x)."""
    lib, dt = _native.lib(), _DT[x.dtype]
    cols = _out_cols(N, act, "linear_q8")
    y = torch.empty(x.shape[:-1] + (cols,), dtype=x.dtype, device=x.device)
    b = None if bias is None else bias.data_ptr()
    out = (y.data_ptr(), dt, cols, M, N, K, _raw_stream(x.device.index))
    if weights == _native.Q8_I8:
        status = lib.psq_gemm_i8_act(q.data_ptr(), K, scale.data_ptr(), w, K, w_scale, b, dt, act, *out)
    elif weights == _native.Q8_E4M3:
        status = lib.psq_gemm_fp8_act(q.data_ptr(), K, scale.data_ptr(), w, K, w_scale, per_row, b, dt, act, *out)
    else:
        status = lib.psq_gemm_fp8_e5m2w(q.data_ptr(), K, scale.data_ptr(), w, K, w_scale, per_row, b, dt, *out)
    return None if status else y


def linear_w4a16_direct(x, M, K, wq, w_scale, w_zero, group_size, N, bias, into=None):
    """x [..., K] contiguous bf16/f16; wq, w_scale, w_zero: device addresses.  [..., N]; into: [M, N]
    rows of x's dtype that take the result."""
    lib, dt, stream = _native.lib(), _DT[x.dtype], _raw_stream(x.device.index)
    ws, nb = _workspace(x.device, stream or None, lib.psq_gemm_wonly_workspace_bytes(_native.W_UINT4, K, M, N, K, group_size))
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device) if into is None else into
    status = lib.psq_gemm_w4a16_ws(x.data_ptr(), dt, K, wq, w_scale, w_zero, group_size,
                                   None if bias is None else bias.data_ptr(), dt, y.data_ptr(), dt, N, M, N, K,
                                   None if ws is None else ws.data_ptr(), nb, stream)
    return None if status else y


# Flags of linear_w8a16 in pinned host memory, each with the last ticket handed out: the kernel stores
# the ticket there when it finds a NaN or Inf, and the host reads it after waiting for the stream -- no
# device-to-host copy.  The store does not keep a larger ticket, so a flag serves one call at a time: a
# call takes one that no call holds and gives it back once its stream was waited for (a call that
# failed in between keeps it: its kernel may still write there).  {device index: (all, free)}; a device
# has as many as calls ran on it at once, at most _MAX_FLAGS, and a call without one takes the separate
# ops.
_host_flags = {}
_MAX_FLAGS = 64
_flags_lock = threading.Lock()


def _take_flag(index):
    """[flag tensor, last ticket, flag word, the list it goes back to]"""
    try:
        return _host_flags[index][1].pop()   # (pop and append are one step each: no lock)
    except (KeyError, IndexError):
        pass
    with _flags_lock:
        made, free = _host_flags.setdefault(index, ([], []))
        if len(made) >= _MAX_FLAGS:
            return None
        flag = torch.zeros(1, dtype=torch.int64, pin_memory=True)
        made.append([flag, 0, ctypes.c_uint64.from_address(flag.data_ptr()), free])
        return made[-1]


def linear_w8a16_launch(x, M, K, wq, w_scale, rot_group, N, bias):
    """Int8Linear's launches: x [..., K] and wq [N, K] contiguous, x f16/bf16, w_scale [N] fp32.
    ([..., N], the check that linear_w8a16_finite answers), or None without a flag."""
    lib, dt, device = _native.lib(), _DT[x.dtype], x.device
    stream = _raw_stream(device.index)
    ws, nb = _workspace(device, stream or None, lib.psq_gemm_wonly_workspace_bytes(_native.W_INT8, K, M, N, K, 0))
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=device)
    rotated = torch.empty(M, K, dtype=x.dtype, device=device) if rot_group else None
    entry = _take_flag(device.index)
    if entry is None:
        return None
    entry[1] = ticket = entry[1] + 1
    try:
        _native.check(lib.psq_linear_w8a16(
            x.data_ptr(), dt, K, rot_group, wq.data_ptr(), w_scale.data_ptr(), None if bias is None else bias.data_ptr(), dt,
            y.data_ptr(), N, M, N, K, None if rotated is None else rotated.data_ptr(),
            None if ws is None else ws.data_ptr(), nb, entry[0].data_ptr(), ticket, stream), "linear_w8a16")
    except Exception:   # refused: the GEMM was not launched
        entry[3].append(entry)
        raise
    return y, (device, entry, ticket)


def linear_w8a16_finite(check):
    """Whether every output of the launch is finite, after waiting for the stream.  An error that the
    wait reports (of this work or of earlier work on the stream) is the caller's."""
    device, entry, ticket = check
    torch.cuda.current_stream(device).synchronize()
    finite = entry[2].value < ticket
    entry[3].append(entry)
    return finite


def linear_w8a16_direct(x, M, K, wq, w_scale, rot_group, N, bias):
    """Launch and check: ([..., N], whether every output is finite), or None (1024 x 5120 x 5120 107.6 ->
    92.0 us a forward, against rotate, GEMM, flag and read-back as separate calls)."""
    done = linear_w8a16_launch(x, M, K, wq, w_scale, rot_group, N, bias)
    return None if done is None else (done[0], linear_w8a16_finite(done[1]))


def direct_available():
    """Whether the direct calls may stand in for the ops: no launch is being timed by name."""
    return _timer is None and _raw_stream is not None


# ------------------------------------------------------------------ dequantize
def dequant_uint4(wq, w_scale, w_zero, group_size, out_dtype=torch.bfloat16):
    _need_gpu(wq, w_scale, w_zero)
    wq = wq.contiguous()
    N, K = wq.shape[0], wq.shape[1] * 2
    out = torch.empty(N, K, dtype=out_dtype, device=wq.device)
    _launch("dequant_uint4", _native.lib().psq_dequant_uint4, _p(wq), _p(w_scale.to(torch.float16).contiguous()),
                                                  _p(w_zero.to(torch.float16).contiguous()), int(group_size), N, K,
                                                  _p(out), _dt(out, "out"), _stream(wq))
    return out


def dequant_i8_rows(q, w_scale, rot_group=0, out_dtype=torch.bfloat16):
    _need_gpu(q, w_scale)
    if not q.is_contiguous():
        q = q.contiguous()
    if w_scale.dtype is not torch.float32 or not w_scale.is_contiguous():
        w_scale = w_scale.to(torch.float32).contiguous()
    N, K = q.shape
    if w_scale.numel() != N:
        raise ValueError(f"dequant_i8_rows: {w_scale.numel()} scales for {N} rows")
    out = torch.empty((N, K), dtype=out_dtype, device=q.device)
    _call("dequant_i8_rows", _native.lib().psq_dequant_i8_rows, q.data_ptr(), w_scale.data_ptr(), N, K, int(rot_group or 0),
          out.data_ptr(), _dt(out, "out"), _raw(q.get_device()))
    return out


def dequant_fp8(q, w_scale, out_dtype=torch.bfloat16, e5m2=None):
    """fp8 weight codes [N, K] times the scale (one, or one per row).  e5m2: the codes are
    float8_e5m2 (default: from q's dtype; uint8 views are e4m3fn)."""
    _need_gpu(q)
    if e5m2 is None:
        e5m2 = q.dtype == torch.float8_e5m2
    q = q.contiguous()
    N, K = q.shape
    s = w_scale.to(device=q.device, dtype=torch.float32).reshape(-1).contiguous()
    out = torch.empty(N, K, dtype=out_dtype, device=q.device)
    name, fn = ("dequant_e5m2", _native.lib().psq_dequant_e5m2) if e5m2 else ("dequant_fp8", _native.lib().psq_dequant_fp8)
    _launch(name, fn, _p(q), _p(s), int(s.numel() > 1), N, K, _p(out), _dt(out, "out"), _stream(q))
    return out


# ------------------------------------------------------------------ text decoder
# What a decoder layer does between its quantized linears.  At one token the host call is most of the time.
# Arguments that need nothing done to them go through _native.direct(), None from there means that they are not
# such and the checks below see to them; those are written out flat, and addresses go to the library as
# integers.  Host us a call, general path and direct: add_rms_norm 11.0 and 6.0, kv_write 7.6 and 3.5, kv_read
# 9.7 and 5.5, paged_attention 10.4 and 5.0 (the launch is 3 of each, an allocation in Python 1.3).
CODES = {None: _native.CODES_NONE, "none": _native.CODES_NONE, "int8": _native.CODES_I8, "fp8": _native.CODES_E4M3}
_CODE_DTYPES = {torch.int8: _native.CODES_I8, torch.float8_e4m3fn: _native.CODES_E4M3,
                torch.bfloat16: _native.CODES_NONE, torch.float16: _native.CODES_NONE}
_HALF = {torch.bfloat16: _native.BF16, torch.float16: _native.F16}
_ROW_DTYPES = (None, torch.int8, torch.float8_e4m3fn)   # of codes


def _elsewhere(name, *tensors):
    raise RuntimeError(f"{name}: psquant kernels need tensors of one GPU (got "
                       f"{', '.join(str(t.device) for t in tensors if t is not None)})")


def add_rms_norm(x, weight, eps=1e-6, residual=None, codes=None, rot_group=0, static_scale=None):
    """RMS norm of h = x + residual (rounded to x's dtype), rows as the operand of gemm_i8 / gemm_fp8.

    x, residual: [M, K] bf16/f16 on the GPU, K a multiple of 16 up to 32768; weight: [K] bf16/f16/f32.
    codes: None (rows in x's dtype), "int8" or "fp8" (e4m3fn); rot_group: ConvRot, as quantize_rows;
    static_scale: fp32 tensor with one element in the place of the rows' own scales.
    Returns (rows [M, K], scale [M] fp32 or None, h or None when there is no residual).
    """
    index = x.get_device()
    if static_scale is None and index >= 0 and _timer is None and (direct := _native.direct()):
        done = direct.add_rms_norm(x, weight, eps, residual, CODES.get(codes, -1), rot_group or 0, _raw(index))
        if done is not None:
            return done
    if index < 0 or weight.get_device() != index or (residual is not None and residual.get_device() != index):
        _elsewhere("add_rms_norm", x, weight, residual)
    code, dtype = CODES.get(codes), x.dtype
    dt = _HALF.get(dtype)
    if code is None:
        raise ValueError(f"add_rms_norm: unknown codes {codes!r}")
    if dt is None:
        raise TypeError(f"add_rms_norm: rows must be bf16/f16, got {dtype}")
    if x.dim() != 2:
        raise ValueError(f"add_rms_norm: rows must be [M, K], got {tuple(x.shape)}")
    M, K = x.shape
    if weight.numel() != K:
        raise ValueError(f"add_rms_norm: weight has {weight.numel()} elements, expected {K}")
    if not x.is_contiguous() or x.data_ptr() % 16 or K % 8:
        x = _rows2d(x)
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = torch.empty(K, dtype=weight.dtype, device=weight.device).copy_(weight.reshape(-1))
    device, h, ldr = x.device, None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype is not dtype:
            raise ValueError(f"add_rms_norm: residual {tuple(residual.shape)} {residual.dtype} does not match the rows")
        if not residual.is_contiguous() or residual.data_ptr() % 16 or K % 8:
            residual = _rows2d(residual)
        ldr = residual.stride(0)
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
    out = torch.empty((M, K), dtype=_ROW_DTYPES[code] or dtype, device=device)
    scale = torch.empty((M,), dtype=torch.float32, device=device) if code else None
    if static_scale is not None:
        if not code:
            raise ValueError("add_rms_norm: a static scale needs codes")
        static_scale = static_scale.to(device=device, dtype=torch.float32).reshape(-1)[:1].contiguous()
    _call("add_rms_norm", _native.lib().psq_add_rms_norm, code, x.data_ptr(), dt, x.stride(0),
          None if residual is None else residual.data_ptr(), ldr, weight.data_ptr(), _dt(weight, "weight"), eps,
          None if h is None else h.data_ptr(), K, int(rot_group or 0), None if static_scale is None else static_scale.data_ptr(),
          out.data_ptr(), K, scale.data_ptr() if code else None, M, K, _raw(index))
    return out, scale, h


def _pools_error(name, k_cache, v_cache, k_scale, v_scale):
    """Raises what is wrong with a paged cache's pools."""
    if _CODE_DTYPES.get(k_cache.dtype) is None or v_cache.dtype is not k_cache.dtype:
        raise TypeError(f"{name}: unsupported cache dtypes {k_cache.dtype}, {v_cache.dtype}")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"{name}: the pools must both be [pages, kv heads, page size, head dim], got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{name}: the pools must be contiguous")
    if _CODE_DTYPES[k_cache.dtype] == _native.CODES_NONE:
        raise ValueError(f"{name}: a 16-bit cache has no scales")
    if k_scale is None or v_scale is None:
        raise ValueError(f"{name}: a cache of codes needs its scales")
    raise ValueError(f"{name}: scales must be contiguous fp32 [pages, kv heads, page size] on the pools' GPU")


def _pools(name, index, k_cache, v_cache, k_scale, v_scale):
    """(codes, pools' shape, scales' addresses) of a paged cache on GPU `index`, checked."""
    if k_cache.get_device() != index or v_cache.get_device() != index or index < 0:
        _elsewhere(name, k_cache, v_cache)
    kind, shape = k_cache.dtype, k_cache.shape
    code = _CODE_DTYPES.get(kind)
    if (code is None or v_cache.dtype is not kind or len(shape) != 4 or v_cache.shape != shape or not k_cache.is_contiguous()
            or not v_cache.is_contiguous()):
        _pools_error(name, k_cache, v_cache, k_scale, v_scale)
    if not code:
        if k_scale is not None or v_scale is not None:
            _pools_error(name, k_cache, v_cache, k_scale, v_scale)
        return code, shape, None, None
    if (k_scale is None or v_scale is None or k_scale.shape != shape[:3] or v_scale.shape != shape[:3]
            or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or not k_scale.is_contiguous()
            or not v_scale.is_contiguous() or k_scale.get_device() != index or v_scale.get_device() != index):
        _pools_error(name, k_cache, v_cache, k_scale, v_scale)
    return code, shape, k_scale.data_ptr(), v_scale.data_ptr()


def _slots(name, slots, index, T=None):
    """slots' address (and the tensor that has it), checked: int64 [tokens] on GPU `index`."""
    if slots.get_device() != index:
        _elsewhere(name, slots)
    if slots.dim() != 1 or slots.dtype is not torch.int64 or (T is not None and slots.shape[0] != T):
        raise ValueError(f"{name}: slots must be int64 [tokens], got {slots.dtype} {tuple(slots.shape)}")
    return slots if slots.is_contiguous() else slots.contiguous()


def _heads(t):
    """(t, token stride, head stride) of [tokens, heads, dim] with unit element stride and 16-byte aligned
    heads: t itself or a packed copy."""
    a, b, c = t.stride()
    if c != 1 or (a | b) & 7 or t.data_ptr() & 15:
        t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
        a, b, c = t.stride()
    return t, a, b


def kv_write(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    """Writes new tokens' keys and values into a paged cache, quantized when the pools hold codes.

    k, v: [tokens, kv heads, head dim] bf16/f16, any token and head strides.  slots: [tokens] int64,
    distinct; slot s is place s % page_size of page s // page_size, a negative slot is skipped.
    k_cache, v_cache: [pages, kv heads, page size, head dim], of k's dtype, int8 or float8_e4m3fn;
    k_scale, v_scale: [pages, kv heads, page size] fp32 for codes (scale = max|row| / 127 or / 448).
    """
    index = k.get_device()
    if index >= 0 and _timer is None and (direct := _native.direct()):
        if direct.kv_write(k, v, slots, k_cache, v_cache, k_scale, v_scale, _raw(index)):
            return
    code, (pages, H, page, D), ks, vs = _pools("kv_write", index, k_cache, v_cache, k_scale, v_scale)
    if v.get_device() != index:
        _elsewhere("kv_write", k, v)
    dtype, shape = k.dtype, k.shape
    dt = _HALF.get(dtype)
    if dt is None or v.dtype is not dtype or (not code and k_cache.dtype is not dtype):
        raise TypeError(f"kv_write: keys {dtype} and values {v.dtype} do not fit a {k_cache.dtype} cache")
    if len(shape) != 3 or v.shape != shape or shape[1] != H or shape[2] != D:
        raise ValueError(f"kv_write: keys {tuple(shape)} and values {tuple(v.shape)} must be [tokens, {H}, {D}]")
    T = shape[0]
    slots = _slots("kv_write", slots, index, T)
    k, k_token, k_head = _heads(k)
    v, v_token, v_head = _heads(v)
    _call("kv_write", _native.lib().psq_kv_write, code, k.data_ptr(), v.data_ptr(), dt, k_token, k_head, v_token, v_head,
          slots.data_ptr(), T, H, D, k_cache.data_ptr(), v_cache.data_ptr(), ks, vs, pages, page, _raw(index))


def rope_kv_write(q, k, v, positions, inv_freq, slots, k_cache, v_cache, k_scale=None, v_scale=None, axes=None, interleaved=False):
    """kv_write of keys turned to their positions, and the turned queries [tokens, heads, head dim].

    q: [tokens, heads, head dim], k, v, slots and the pools as in kv_write.  inv_freq: [pairs] float64 (other
    types are converted on each call), the angle per position of each pair, pairs a multiple of 8; pair i is
    the elements i and i + pairs of a row, 2 i and 2 i + 1 when interleaved; elements from 2 * pairs on stay as
    they are.  positions: [tokens] int32 or int64, or [n, tokens] with axes, [pairs] int32: which of the n
    positions (time, height and width, say) turns each pair.  Angles are worked out in fp64 and sines in fp32 (off by at
    most 2^-22 + 3 |angle| 2^-53); keys are turned in fp32 and quantized from there.
    """
    index = q.get_device()
    if index >= 0 and _timer is None and (direct := _native.direct()):
        done = direct.rope_kv_write(q, k, v, positions, inv_freq, slots, k_cache, v_cache, k_scale, v_scale, axes, interleaved, _raw(index))
        if done is not None:
            return done
    code, (pages, H, page, D), ks, vs = _pools("rope_kv_write", index, k_cache, v_cache, k_scale, v_scale)
    for t in (k, v, positions, inv_freq) + (() if axes is None else (axes,)):
        if t.get_device() != index:
            _elsewhere("rope_kv_write", q, t)
    dtype, shape = q.dtype, k.shape
    dt = _HALF.get(dtype)
    if dt is None or k.dtype is not dtype or v.dtype is not dtype or (not code and k_cache.dtype is not dtype):
        raise TypeError(f"rope_kv_write: queries {dtype}, keys {k.dtype} and values {v.dtype} do not fit a {k_cache.dtype} cache")
    if len(shape) != 3 or v.shape != shape or shape[1] != H or shape[2] != D:
        raise ValueError(f"rope_kv_write: keys {tuple(shape)} and values {tuple(v.shape)} must be [tokens, {H}, {D}]")
    T = shape[0]
    if q.dim() != 3 or q.shape[0] != T or q.shape[2] != D:
        raise ValueError(f"rope_kv_write: queries {tuple(q.shape)} must be [{T}, heads, {D}]")
    if inv_freq.dim() != 1 or not 0 < 2 * inv_freq.shape[0] <= D or inv_freq.shape[0] % 8:
        raise ValueError(f"rope_kv_write: inv_freq {tuple(inv_freq.shape)} must have a multiple of 8 pairs, at most {D // 2}")
    pairs = inv_freq.shape[0]
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape[-1:] != (T,) or positions.dim() != (1 if axes is None else 2):
        raise ValueError(f"rope_kv_write: positions must be int32 or int64 [{T}], or [n, {T}] with axes, got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    if axes is not None and (axes.dtype is not torch.int32 or axes.shape != (pairs,) or positions.shape[0] == 0):
        raise ValueError(f"rope_kv_write: axes must be int32 [{pairs}] for one row of positions or more")
    slots = _slots("rope_kv_write", slots, index, T)
    if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    if axes is not None and not axes.is_contiguous():
        axes = axes.contiguous()
    q, q_token, q_head = _heads(q)
    k, k_token, k_head = _heads(k)
    v, v_token, v_head = _heads(v)
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    _call("rope_kv_write", _native.lib().psq_rope_kv_write, code, q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, q_token, q_head, k_token,
          k_head, v_token, v_head, positions.data_ptr(), 64 if positions.dtype is torch.int64 else 32,
          1 if axes is None else positions.shape[0], 0 if axes is None else positions.stride(0), None if axes is None else axes.data_ptr(),
          inv_freq.data_ptr(), 2 * pairs, int(bool(interleaved)), slots.data_ptr(), T, q.shape[1], H, D, k_cache.data_ptr(),
          v_cache.data_ptr(), ks, vs, pages, page, out.data_ptr(), _raw(index))
    return out


def kv_read(slots, k_cache, v_cache, k_scale=None, v_scale=None, out_dtype=None):
    """Cached tokens back as dense rows: (k, v), each [tokens, kv heads, head dim] of out_dtype (default: the
    cache's dtype, bf16 for codes).  slots as in kv_write; a negative slot reads as zeros."""
    index = slots.get_device()
    if out_dtype is None:
        out_dtype = torch.bfloat16 if _CODE_DTYPES.get(k_cache.dtype) else k_cache.dtype
    if index >= 0 and _timer is None and (direct := _native.direct()):
        done = direct.kv_read(slots, k_cache, v_cache, k_scale, v_scale, _DT.get(out_dtype, -1), _raw(index))
        if done is not None:
            return done
    code, (pages, H, page, D), ks, vs = _pools("kv_read", index, k_cache, v_cache, k_scale, v_scale)
    dt = _DT.get(out_dtype)
    if dt is None:
        raise TypeError(f"kv_read: unsupported dtype {out_dtype}")
    slots = _slots("kv_read", slots, index)
    T = slots.shape[0]
    k = torch.empty((T, H, D), dtype=out_dtype, device=slots.device)
    v = torch.empty_like(k)
    _call("kv_read", _native.lib().psq_kv_read, code, slots.data_ptr(), T, k_cache.data_ptr(), v_cache.data_ptr(),
          0 if code else _HALF[k_cache.dtype], ks, vs, pages, page, H, D, k.data_ptr(), v.data_ptr(), dt, _raw(index))
    return k, v


def paged_attention(q, k_cache, v_cache, block_table, lengths, k_scale=None, v_scale=None, scale=None, window=0,
                    max_len=None, return_lse=False, sinks=0):
    """Attention of one new token per sequence over a paged cache: [batch, heads, head dim] of q's dtype.

    q: [batch, heads, head dim] bf16/f16, heads a multiple of the cache's kv heads; a 16-bit cache has q's
    dtype.  block_table: [batch, columns] int32, the page of token t in column t // page_size; lengths:
    [batch] int32, each sequence's tokens, the new one included (0: zeros).  scale: of the scores (default
    head_dim ** -0.5); window: the last tokens that are attended to (0: all); sinks: the first tokens of a
    sequence that a window does not hide.  max_len: about the longest
    length, for the number of workgroups (default: what the table can hold; any value gives right results).
    return_lse: also the natural log of the softmax's denominator, [batch, heads] fp32.
    A sequence that needs a page outside the pool, or more tokens than its table has, gets NaN.
    """
    index = q.get_device()
    if index >= 0 and _timer is None and (direct := _native.direct()):
        raw = _raw(index)
        done = direct.paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scale, window, max_len, return_lse,
                                      _workspaces.get((index, raw or None)), raw, sinks)
        if done is not None:
            return done
    code, (pages, Hk, page, D), ks, vs = _pools("paged_attention", index, k_cache, v_cache, k_scale, v_scale)
    if block_table.get_device() != index or lengths.get_device() != index:
        _elsewhere("paged_attention", q, block_table, lengths)
    dtype, shape = q.dtype, q.shape
    dt = _HALF.get(dtype)
    if dt is None or (not code and k_cache.dtype is not dtype):
        raise TypeError(f"paged_attention: {dtype} queries do not fit a {k_cache.dtype} cache")
    if len(shape) != 3 or shape[2] != D or shape[1] % Hk:
        raise ValueError(f"paged_attention: queries {tuple(shape)} must be [batch, a multiple of {Hk}, {D}]")
    B, H, _ = shape
    if block_table.dim() != 2 or block_table.dtype is not torch.int32 or block_table.shape[0] != B:
        raise ValueError(f"paged_attention: block_table must be int32 [{B}, columns]")
    if lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.shape[0] != B:
        raise ValueError(f"paged_attention: lengths must be int32 [{B}]")
    if window is None or window < 0:
        raise ValueError("paged_attention: window must be 0 or more")
    if sinks is None or sinks < 0 or (sinks and not window):
        raise ValueError("paged_attention: sinks must be 0 or more, with a window")
    cols = block_table.shape[1]
    if not block_table.is_contiguous() and cols > 1 and block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    q, q_batch, q_head = _heads(q)
    max_len = cols * page if max_len is None or max_len < 0 else min(int(max_len), cols * page)
    if window and window + sinks < max_len:
        max_len = int(window + sinks)
    lib, raw, device = _native.lib(), _raw(index), q.device
    out = torch.empty((B, H, D), dtype=dtype, device=device)
    lse = torch.empty((B, H), dtype=torch.float32, device=device) if return_lse else None
    nb = lib.psq_paged_attention_workspace_bytes(code, B, H, Hk, D, max_len)
    if nb > 0 and lib.psq_paged_attention_own_workspace(code, B, H, Hk, D, max_len):
        ws = torch.empty(nb, dtype=torch.uint8, device=device)   # two launches: the call's own
    else:
        ws, nb = _workspace(device, raw or None, nb)
    _call("paged_attention", lib.psq_paged_attention_sinks if sinks else lib.psq_paged_attention, code, q.data_ptr(), dt, q_batch,
          q_head, k_cache.data_ptr(), v_cache.data_ptr(), ks, vs, pages, page, block_table.data_ptr(), block_table.stride(0), cols,
          lengths.data_ptr(), B, H, Hk, D, D ** -0.5 if scale is None else scale, window, *((sinks,) if sinks else ()), max_len, out.data_ptr(),
          lse.data_ptr() if return_lse else None, None if ws is None else ws.data_ptr(), nb, raw)
    return (out, lse) if return_lse else out


def _rows_on_cache(name, q, rows, k_cache, v_cache, block_table, lengths, k_scale, v_scale, window, sinks, *others):
    """Checked arguments that the attention of prompts and of trees have in common; rows: q's dims in front of [heads, dim]."""
    index = q.get_device()
    code, (pages, Hk, page, D), ks, vs = _pools(name, index, k_cache, v_cache, k_scale, v_scale)
    for t in (block_table, lengths) + others:
        if t.get_device() != index:
            _elsewhere(name, q, t)
    dt = _HALF.get(q.dtype)
    if dt is None or (not code and k_cache.dtype is not q.dtype):
        raise TypeError(f"{name}: {q.dtype} queries do not fit a {k_cache.dtype} cache")
    if q.dim() != rows + 2 or q.shape[-1] != D or q.shape[-2] % Hk:
        raise ValueError(f"{name}: queries {tuple(q.shape)} must be [{'tokens' if rows == 1 else 'batch, drafts'}, a multiple of {Hk}, {D}]")
    if lengths.dtype is not torch.int32 or lengths.dim() != 1:
        raise ValueError(f"{name}: lengths must be int32 [batch]")
    B = lengths.shape[0]
    if block_table.dim() != 2 or block_table.dtype is not torch.int32 or block_table.shape[0] != B:
        raise ValueError(f"{name}: block_table must be int32 [{B}, columns]")
    if window is None or window < 0 or sinks is None or sinks < 0 or (sinks and not window):
        raise ValueError(f"{name}: window and sinks must be 0 or more, sinks with a window")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    return index, code, dt, (pages, Hk, page, D), ks, vs, block_table, lengths if lengths.is_contiguous() else lengths.contiguous()


def _parts(code, rows, B, N, H, Hk, D, window, sinks, max_len, device):
    """(memory of the call's own for the parts of split sequences, its bytes)."""
    nb = _native.lib().psq_paged_block_workspace_bytes(code, rows, B, N, H, Hk, D, window, sinks, max_len)
    return (torch.empty(nb, dtype=torch.uint8, device=device) if nb else None), nb


def paged_prompt_attention(q, k_cache, v_cache, block_table, starts, lengths, k_scale=None, v_scale=None, scale=None, window=0, sinks=0,
                           max_len=None, return_lse=False):
    """Attention of a batch of prompts, or of parts of them, over the paged cache that holds them: [tokens, heads, dim].

    q: [tokens, heads, head dim] bf16/f16; rows starts[b] .. starts[b + 1] - 1 are the newest tokens of sequence b, its
    last ones.  starts: [batch + 1] int32 from 0, not decreasing; rows from the last one on get zeros.  lengths: [batch]
    int32, the new tokens included.  A token sees those in front of it and itself; with a window, of these the last
    `window` and the first `sinks` of the sequence.  The cache, scale, max_len and return_lse (lse [tokens, heads]) as
    in paged_attention.
    Scores, softmax statistics and sums are fp32; a probability meets its value as one 16-bit number, of q's type or bf16 on
    codes, off by half a step as the output is (f16 rows on codes: as two; paged_attention: as two always).
    A row that sees a token whose page is outside the pool, or past the table, gets NaN.
    """
    if (index := q.get_device()) >= 0 and _timer is None and (direct := _native.direct()):
        done = direct.paged_prompt_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, starts, None, scale, window, sinks,
                                          max_len, return_lse, _raw(index))
        if done is not None:
            return done
    name = "paged_prompt_attention"
    index, code, dt, (pages, Hk, page, D), ks, vs, block_table, lengths = _rows_on_cache(
        name, q, 1, k_cache, v_cache, block_table, lengths, k_scale, v_scale, window, sinks, starts)
    (T, H, _), B, cols = q.shape, lengths.shape[0], block_table.shape[1]
    if starts.dtype is not torch.int32 or starts.shape != (B + 1,):
        raise ValueError(f"{name}: starts must be int32 [{B + 1}]")
    if not starts.is_contiguous():
        starts = starts.contiguous()
    q, q_token, q_head = _heads(q)
    max_len = cols * page if max_len is None or max_len < 0 else min(int(max_len), cols * page)
    out = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, H), dtype=torch.float32, device=q.device) if return_lse else None
    ws, nb = _parts(code, T, B, 0, H, Hk, D, window, sinks, max_len, q.device)
    _call(name, _native.lib().psq_paged_prompt_attention, code, q.data_ptr(), dt, q_token, q_head, k_cache.data_ptr(), v_cache.data_ptr(),
          ks, vs, pages, page, block_table.data_ptr(), block_table.stride(0), cols, starts.data_ptr(), lengths.data_ptr(), B, T, H, Hk, D,
          D ** -0.5 if scale is None else scale, window, sinks, max_len, out.data_ptr(), lse.data_ptr() if return_lse else None,
          None if ws is None else ws.data_ptr(), nb, _raw(index))
    return (out, lse) if return_lse else out


def paged_tree_attention(q, k_cache, v_cache, block_table, lengths, parents, k_scale=None, v_scale=None, drafts=None, scale=None,
                         window=0, sinks=0, max_len=None, return_lse=False):
    """Attention of a tree of drafted tokens per sequence over the paged cache that holds them: [batch, n, heads, dim].

    q: [batch, n, heads, head dim] bf16/f16, n up to 64.  The last n tokens of a sequence (of its length, lengths[b]) are its
    drafts, draft i at place lengths[b] - n + i of the cache; drafts: [batch] int32, how many of the n there are
    (in place of n; rows past them get zeros).  parents: [batch, n] int32: the draft that each one goes on from, an
    earlier one, or -1 (every other value means that too): the text in front.  A draft sees that text, the drafts on its
    way from there and itself.  Its position is the text's length plus the number of drafts in front of it on its way;
    window and sinks count positions.  The rest as in paged_prompt_attention (lse [batch, n, heads]).
    """
    if (index := q.get_device()) >= 0 and _timer is None and (direct := _native.direct()):
        done = direct.paged_tree_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, parents, drafts, scale, window, sinks,
                                         max_len, return_lse, _raw(index))
        if done is not None:
            return done
    name = "paged_tree_attention"
    index, code, dt, (pages, Hk, page, D), ks, vs, block_table, lengths = _rows_on_cache(
        name, q, 2, k_cache, v_cache, block_table, lengths, k_scale, v_scale, window, sinks, parents, *(() if drafts is None else (drafts,)))
    (B, N, H, _), cols = q.shape, block_table.shape[1]
    if lengths.shape[0] != B or parents.dtype is not torch.int32 or parents.shape != (B, N):
        raise ValueError(f"{name}: lengths and parents must be int32 [{B}] and [{B}, {N}]")
    if N > 64:
        raise ValueError(f"{name}: {N} drafts, at most 64")
    if drafts is not None and (drafts.dtype is not torch.int32 or drafts.shape != (B,)):
        raise ValueError(f"{name}: drafts must be int32 [{B}]")
    if not parents.is_contiguous():
        parents = parents.contiguous()
    if drafts is not None and not drafts.is_contiguous():
        drafts = drafts.contiguous()
    q, q_token, q_head = _heads(q.reshape(B * N, H, D))
    max_len = cols * page if max_len is None or max_len < 0 else min(int(max_len), cols * page)
    out = torch.empty((B, N, H, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, N, H), dtype=torch.float32, device=q.device) if return_lse else None
    ws, nb = _parts(code, B * N, B, N, H, Hk, D, window, sinks, max_len, q.device)
    _call(name, _native.lib().psq_paged_tree_attention, code, q.data_ptr(), dt, q_token, q_head, k_cache.data_ptr(), v_cache.data_ptr(),
          ks, vs, pages, page, block_table.data_ptr(), block_table.stride(0), cols, lengths.data_ptr(), parents.data_ptr(),
          None if drafts is None else drafts.data_ptr(), B, N, H, Hk, D, D ** -0.5 if scale is None else scale, window, sinks, max_len,
          out.data_ptr(), lse.data_ptr() if return_lse else None,
          None if ws is None else ws.data_ptr(), nb, _raw(index))
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ checks
# Non-finite flags, one per (device, stream), with the last ticket handed out: a call raises the
# flag to its ticket when it finds a NaN or Inf, and the flag is never cleared.
_nonfinite = {}


def any_nonfinite(t):
    """True when the CUDA tensor t (bf16 / f16 / f32) holds a NaN or an Inf: one pass over t and an
    8-byte read back (a synchronization, as `not torch.isfinite(t).all()`, which this replaces where
    it is checked on every call)."""
    _need_gpu(t)
    t = t.contiguous()
    stream = _stream(t)
    key = (t.device.index, stream.value)
    entry = _nonfinite.get(key)
    if entry is None:
        entry = _nonfinite[key] = [torch.zeros(1, dtype=torch.int64, device=t.device), 0]
    entry[1] += 1
    _launch("flag_nonfinite", _native.lib().psq_flag_nonfinite, _p(t), _dt(t, "t"), t.numel(), _p(entry[0]),
            entry[1], stream)
    return int(entry[0].item()) >= entry[1]


def device_supported(device):
    device = torch.device(device)
    if device.type != "cuda":
        return False
    index = device.index if device.index is not None else torch.cuda.current_device()
    return bool(_native.lib().psq_device_supported(index))
