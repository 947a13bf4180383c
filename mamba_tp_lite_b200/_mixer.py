"""Kernel driver shared by the dense and tensor-parallel mixers.

One mixer forward is this chain of libmtp calls (T = batch x positions):

  prefill (T >= 1):
    in_proj   GEMM            xn [T,D] -> xz [T,2Es]                 (tp_model.py:91)
    conv1d    conv1d+SiLU     xz -> xc [T,Es] (input of x_proj)      (tp_model.py:95-100)
    x_proj    GEMM            xc -> partial [T,R+2N] fp32            (tp_model.py:106)
    AR #1     reduce_xproj    partial -> dt_low [T,R], B|C [T,2N]    (tp_model.py:107-108)
    dt_proj   GEMM+softplus   dt_low -> dt [T,Es] model dtype        (tp_model.py:110-111)
    scan      scan over xc + D skip + SiLU(z) gate -> y [T,Es], final conv/ssm state (tp_model.py:101-129)
    out_proj  GEMM            y -> partial [T,D] fp32                (tp_model.py:131)
    AR #2     reduce_outproj  partial -> resid += out; normed = RMSNorm_next(resid)
                                                                      (tp_model.py:132-134, :254-257)
  step (one token per sequence):
    in_proj GEMV, conv1d+SiLU (pure), x_proj GEMV, AR #1, then one in-place step kernel
    (conv shift, dt_proj, softplus, state update, output, gate), out_proj GEMV, AR #2.

Activations stay in the model dtype; the residual stream, the reduction
partials, dt, B, C and the SSM state are fp32.

A dense mixer with int8 linears (``MambaLM.quantize_linears``) takes its in_proj input
as int8 rows, quantises y in front of out_proj, and hands the out_proj result to
``add_rms_norm_int8`` in fp32; conv1d, x_proj, dt_proj and the scan are as above.
"""
from __future__ import annotations

import os

import torch

from . import _lib as L
from .int8 import Int8Rows, int8_linear, quantize_rows
from .tp_utils import KERNEL_MODES, ROW_MODES, comm_for, count_collective

# Optional launch timing for benchmarks: when set to a dict, CUDA events are
# recorded around the named kernel launches into PROFILE[name] as
# (start_event, end_event, work) with work = algorithmic FLOPs (GEMMs) or bytes (scan).
PROFILE = None

# Set by the LM driver while it runs micro-batches on separate streams
# (_LMKernels._prefill_overlapped): every reduction is then issued on this one
# communication stream, in the host's order, between event waits on the calling
# stream; the driver accounts the collectives itself (full-batch shapes).
OVERLAP_STREAM = None


def _on_comm_stream(fn, tensors) -> None:
    """Runs ``fn`` (which launches on the current stream) on OVERLAP_STREAM after
    the calling stream's work, and makes the calling stream wait for it."""
    cur = torch.cuda.current_stream()
    cs = OVERLAP_STREAM
    cs.wait_stream(cur)
    with torch.cuda.stream(cs):
        fn()
    for t in tensors:
        if t is not None:
            t.record_stream(cs)
    cur.wait_stream(cs)


def _prof_begin():
    if PROFILE is None:
        return None
    e = torch.cuda.Event(enable_timing=True)
    e.record()
    return e


def _prof_end(start, name, work):
    if start is None:
        return
    e = torch.cuda.Event(enable_timing=True)
    e.record()
    PROFILE.setdefault(name, []).append((start, e, work))


class Watched:
    """A weight that int8 rows were made from, so that a later change is noticed: in place (``load_state_dict``, an optimiser;
    not through ``.data`` or of an inference tensor, which torch does not count), by another tensor in its place, or by a
    move to another device or type.  A deep or pickled copy watches the weight that was copied with it."""

    __slots__ = ("weight", "at", "version")

    def __init__(self, w):
        # held, and not by a weak reference, which torch.utils.swap_tensors refuses
        self.weight, self.at = w, w.data_ptr()
        self.version = None if w.is_inference() else w._version

    def changed(self, w) -> bool:
        if w is None or self.weight is not w or w.data_ptr() != self.at:
            return True
        return self.version is not None and w._version != self.version

    def __getstate__(self):
        return (None if self.changed(self.weight) else self.weight,)

    def __setstate__(self, state):
        if state[0] is None:
            self.weight, self.at, self.version = None, 0, None
        else:
            self.__init__(state[0])


class MixerKernels:
    """Mixin holding the kernel calls.  Expects the reference's parameter
    layout on ``self`` (in_proj, conv1d, x_proj, dt_proj, A_log, D, out_proj)
    plus ``cfg``, ``es`` (local channels), ``rank``, ``world_size``, ``group``,
    ``layer_idx``, ``_site_modes`` ({"x_proj": name, "out_proj": name} or None
    for the dense mixer) and ``comm`` (CommCounter) and ``_out_bias()``."""

    _int8 = None  # (in_proj, out_proj) weights as Int8Rows, a scale for each output channel
    _int8_of = None  # what they were made from: a Watched for each that is a parameter, else None

    # ------------------------------------------------------------ helpers
    def _set_int8(self, on: bool) -> None:
        rows = (quantize_rows(self.in_proj.weight), quantize_rows(self.out_proj.weight)) if on else None
        of = tuple(None if w is None else Watched(w) for w in self._int8_parameters()) if on else None
        self._int8, self._int8_of = rows, of

    def _int8_parameters(self):
        modules = self._modules  # past nn.Module's look-up, which would be most of a check
        return modules["in_proj"]._parameters.get("weight"), modules["out_proj"]._parameters.get("weight")

    def _check_int8(self) -> None:
        if self._int8_of is None:
            return
        (i, o), (w_i, w_o) = self._int8_of, self._int8_parameters()
        if i is not None and i.changed(w_i) or o is not None and o.changed(w_o):
            raise RuntimeError(f"layer {self.layer_idx}: the weights of in_proj or out_proj have changed or moved since "
                               "quantize_linears(); call it again")

    def _dt(self) -> torch.dtype:
        return self.in_proj.weight.dtype

    def _gemm(self, a, w, out, epi=L.EPI_STORE, bias=None, tag=None):
        M, K = a.shape
        N = w.shape[0]
        ev = _prof_begin() if tag else None
        L.call("mtp_gemm", L.ptr(a), L.ptr(w), L.ptr(out), M, N, K, a.stride(0), w.stride(0), out.stride(0),
               L.dtype_code(a.dtype), L.dtype_code(out.dtype), epi, L.ptr(bias),
               L.dtype_code(bias.dtype) if bias is not None else 0, L.stream_ptr())
        _prof_end(ev, tag, 2.0 * M * N * K)

    def _in_proj(self, xn, tag):
        """xz = in_proj(xn) in the model dtype; xn [T, D], or its int8 rows for int8 linears."""
        w, bias, dt_ = self.in_proj.weight, self.in_proj.bias, self._dt()
        if isinstance(xn, Int8Rows):
            ev = _prof_begin()
            xz = int8_linear(xn, self._int8[0], None if bias is None else bias.detach(), dtype=dt_)
            _prof_end(ev, tag, 2.0 * xz.numel() * w.shape[1])
            return xz
        xz = torch.empty(xn.shape[0], 2 * self.es, device=xn.device, dtype=dt_)
        self._gemm(xn, w, xz, *((L.EPI_BIAS, bias) if bias is not None else (L.EPI_STORE, None)), tag=tag)
        return xz

    def _out_proj_int8(self, y, tag):
        """out_proj(y) + bias in fp32 through int8 linears: what is added to the residual stream."""
        rows, bias = quantize_rows(y), self._out_bias()
        ev = _prof_begin()
        out = int8_linear(rows, self._int8[1], None if bias is None else bias.detach(), dtype=torch.float32)
        _prof_end(ev, tag, 2.0 * out.numel() * y.shape[1])
        return out

    def _check_input(self, x: torch.Tensor, what: str):
        L.require_cuda(x, what)
        if x.dtype != self._dt():
            raise TypeError(f"{what}: input dtype {x.dtype} != model dtype {self._dt()}")

    def _reduce_x(self, partial, dt_low, bc):
        """AllReduce #1 (tp_model.py:107) fused with the dt / B|C split."""
        cfg = self.cfg
        rows = partial.shape[0]
        name = None if self._site_modes is None else self._site_modes["x_proj"]
        ctx = None
        mode = L.RED_FP32
        if name is not None:
            if OVERLAP_STREAM is None:
                count_collective(self.comm, name, partial.shape, self._dt())
            mode = KERNEL_MODES[name]
            ctx = comm_for(self)

        def launch():
            L.call("mtp_reduce_xproj", ctx, mode, L.ptr(partial), rows, cfg.dt_rank, 2 * cfg.d_state, L.ptr(dt_low),
                   L.dtype_code(dt_low.dtype), L.ptr(bc), L.stream_ptr())

        if OVERLAP_STREAM is not None:
            _on_comm_stream(launch, (partial, dt_low, bc))
        else:
            ev = _prof_begin()
            launch()
            if ev is not None:
                _prof_end(ev, "reduce_x", L.comm_sent_bytes(ctx, mode, rows, partial.shape[1],
                                                            L.dtype_code(dt_low.dtype)))

    def _xproj_fused(self, xc, partial, dt_low, bc) -> bool:
        """x_proj GEMM fused with AllReduce #1 (tp_model.py:106-108): the GEMM's epilogue
        writes the wire rows (or, at world size 1, dt_low | B|C after the wire round trip),
        so the fp32 partial is not written; ``partial`` is only the fallback buffer of the
        library for shapes the fused form does not take.  False (nothing launched) for the
        per-tensor-scale variants and while micro-batches overlap."""
        cfg = self.cfg
        name = None if self._site_modes is None else self._site_modes["x_proj"]
        if OVERLAP_STREAM is not None or (name is not None and name not in ROW_MODES):
            return False
        ctx, mode = None, L.RED_FP32
        if name is not None:
            count_collective(self.comm, name, partial.shape, self._dt())
            mode = KERNEL_MODES[name]
            ctx = comm_for(self)
        T, n_out = partial.shape
        w = self.x_proj.weight
        ev = _prof_begin()
        L.call("mtp_xproj_fused", ctx, mode, L.ptr(xc), xc.stride(0), L.ptr(w), w.stride(0), L.dtype_code(xc.dtype), T,
               n_out, xc.shape[1], cfg.dt_rank, L.ptr(partial), L.ptr(dt_low), L.dtype_code(dt_low.dtype), L.ptr(bc),
               L.stream_ptr())
        _prof_end(ev, "x_proj+reduce_x", 2.0 * T * n_out * xc.shape[1])
        return True

    def _reduce_out(self, partial, resid, norm_w, eps, normed):
        """AllReduce #2 (tp_model.py:132-134) fused with the bias, the block
        residual and the next RMSNorm."""
        rows, d = partial.shape
        name = None if self._site_modes is None else self._site_modes["out_proj"]
        ctx = None
        mode = L.RED_FP32
        if name is not None:
            if OVERLAP_STREAM is None:
                count_collective(self.comm, name, partial.shape, self._dt())
            mode = KERNEL_MODES[name]
            ctx = comm_for(self)
        bias = self._out_bias()
        odt = normed.dtype if normed is not None else self._dt()

        def launch():
            L.call("mtp_reduce_outproj", ctx, mode, L.ptr(partial), rows, d, L.ptr(bias), L.ptr(resid), L.ptr(norm_w),
                   float(eps), L.ptr(normed), L.dtype_code(odt), L.stream_ptr())

        if OVERLAP_STREAM is not None:
            _on_comm_stream(launch, (partial, resid, normed))
        else:
            ev = _prof_begin()
            launch()
            if ev is not None:
                _prof_end(ev, "reduce_out", L.comm_sent_bytes(ctx, mode, rows, d, L.dtype_code(odt)))

    def _fused_dt_ok(self) -> bool:
        """The fused dt_proj + scan kernel (opt-in, MTP_FUSED_DT=1) for bf16 models
        with d_state 16, d_inner per rank divisible by 128 and dt_rank divisible
        by 8.  Off by default: on B200 (32 x 1024 tokens) the dt_proj GEMM plus
        the scan is faster at every shard width: 4096 channels 1.12 vs 1.47 ms,
        2048: 0.64 vs 0.92, 1024: 0.40 vs 0.57, 512: 0.32 vs 0.37."""
        cfg = self.cfg
        return (self._dt() == torch.bfloat16 and cfg.d_state == 16 and cfg.d_conv == 4 and self.es % 128 == 0
                and cfg.dt_rank % 8 == 0 and cfg.dt_rank <= 256 and os.environ.get("MTP_FUSED_DT", "0") == "1")

    # ------------------------------------------------------------ prefill core
    def _prefill_core(self, xn, B, Lq, conv_init, ssm_init, resid, norm_w=None, eps=0.0, normed=None,
                      conv_out=None, ssm_out=None):
        """xn [T, D] (model dtype, RMS-normed block input).  Adds the mixer
        output into ``resid`` [T, D] fp32 and, when ``normed`` is given, writes
        RMSNorm(resid) * norm_w into it.  Returns (conv_final, ssm_final),
        written into ``conv_out`` / ``ssm_out`` when given."""
        g = self._prefill_stages(xn, B, Lq, conv_init, ssm_init, resid, norm_w, eps, normed, conv_out, ssm_out)
        next(g)
        try:
            next(g)
        except StopIteration as done:
            return done.value
        raise RuntimeError("prefill stages did not finish")

    def _prefill_stages(self, xn, B, Lq, conv_init, ssm_init, resid, norm_w=None, eps=0.0, normed=None,
                        conv_out=None, ssm_out=None):
        """_prefill_core as a generator: it yields once, after AllReduce #1 has been
        issued, so a driver can interleave the launches of several micro-batches."""
        cfg = self.cfg
        y, conv_final, ssm_final = yield from self._prefill_mix(self._in_proj(xn, "in_proj"), B, Lq, conv_init, ssm_init,
                                                                conv_out, ssm_out)
        partial_o = torch.empty(xn.shape[0], cfg.d_model, device=xn.device, dtype=torch.float32)
        self._gemm(y, self.out_proj.weight, partial_o, tag="out_proj")
        self._reduce_out(partial_o, resid, norm_w, eps, normed)
        return conv_final, ssm_final

    def _prefill_int8(self, rows, B, Lq, conv_init, ssm_init):
        """rows: int8 rows [T, D] of the block input.  Returns (mixer output fp32 [T, D], conv_final, ssm_final)."""
        g = self._prefill_mix(self._in_proj(rows, "in_proj"), B, Lq, conv_init, ssm_init)
        next(g)
        try:
            next(g)
        except StopIteration as done:
            y, conv_final, ssm_final = done.value
            return self._out_proj_int8(y, "out_proj"), conv_final, ssm_final
        raise RuntimeError("prefill stages did not finish")

    def _prefill_mix(self, xz, B, Lq, conv_init, ssm_init, conv_out=None, ssm_out=None):
        """From in_proj's output xz [T, 2Es] to out_proj's input: (y [T, Es], conv_final, ssm_final), as a generator that
        yields once, after AllReduce #1 has been issued."""
        cfg = self.cfg
        es, n, r, k = self.es, cfg.d_state, cfg.dt_rank, cfg.d_conv
        T = xz.shape[0]
        dt_ = self._dt()
        dev = xz.device
        conv_w = self.conv1d.weight
        conv_b = self.conv1d.bias
        xc = torch.empty(T, es, device=dev, dtype=dt_)
        ev = _prof_begin()
        L.call("mtp_conv1d_silu", L.ptr(xz), 2 * es, L.ptr(conv_w), L.ptr(conv_b), L.ptr(conv_init), L.ptr(xc), es,
               B, Lq, es, k, L.dtype_code(dt_), L.stream_ptr())
        _prof_end(ev, "conv1d", 2 * T * es * xz.element_size())  # x read, xc written
        partial_x = torch.empty(T, r + 2 * n, device=dev, dtype=torch.float32)
        dt_low = torch.empty(T, r, device=dev, dtype=dt_)
        bc = torch.empty(T, 2 * n, device=dev, dtype=torch.float32)
        if not self._xproj_fused(xc, partial_x, dt_low, bc):
            self._gemm(xc, self.x_proj.weight, partial_x, tag="x_proj")
            self._reduce_x(partial_x, dt_low, bc)
        yield
        y = torch.empty(T, es, device=dev, dtype=dt_)
        conv_final = conv_out if conv_out is not None else torch.empty(B, es, k - 1, device=dev, dtype=dt_)
        ssm_final = ssm_out if ssm_out is not None else torch.empty(B, es, n, device=dev, dtype=torch.float32)
        esz = xz.element_size()
        if self._fused_dt_ok():
            # dt_proj + softplus inside the scan kernel (tensor cores); no dt round trip
            ev = _prof_begin()
            L.call("mtp_scan_prefill_fused", L.ptr(xz), 2 * es, L.ptr(dt_low), r, L.ptr(self.dt_proj.weight),
                   L.ptr(self.dt_proj.bias), L.ptr(bc), 2 * n, L.ptr(self.A_log), L.ptr(self.D), L.ptr(conv_w),
                   L.ptr(conv_b), L.ptr(conv_init), L.ptr(ssm_init), L.ptr(y), es, L.ptr(conv_final),
                   L.ptr(ssm_final), B, Lq, es, n, r, k, L.stream_ptr())
            _prof_end(ev, "scan", T * (es * 3 * esz + (r + 2 * n) * 4) + B * es * (2 * n * 4 + 2 * (k - 1) * esz))
            return y, conv_final, ssm_final
        # dt = softplus(dt_proj(dt_low)) in the model dtype, as the reference's dt_proj output
        # (tp_model.py:110-111); the scan widens it to fp32
        dt = torch.empty(T, es, device=dev, dtype=dt_)
        self._gemm(dt_low, self.dt_proj.weight, dt, L.EPI_BIAS_SOFTPLUS, self.dt_proj.bias, tag="dt_proj")
        ev = _prof_begin()
        # the scan reads the conv output xc that x_proj already consumed (no conv recompute)
        L.call("mtp_scan_prefill_xc", L.ptr(xc), es, L.ptr(xz), 2 * es, L.ptr(dt), es, L.dtype_code(dt_), L.ptr(bc),
               2 * n, L.ptr(self.A_log), L.ptr(self.D), L.ptr(conv_init), L.ptr(ssm_init), L.ptr(y), es,
               L.ptr(conv_final), L.ptr(ssm_final), B, Lq, es, n, k, L.dtype_code(dt_), L.stream_ptr())
        # algorithmic bytes: x, z, dt, y in the model dtype, B|C fp32 (+ per-sequence state I/O)
        _prof_end(ev, "scan", T * (es * 4 * esz + 2 * n * 4) + B * es * (2 * n * 4 + 2 * (k - 1) * esz))
        return y, conv_final, ssm_final

    # ------------------------------------------------------------ step core
    def _step_core(self, xn, conv_state, ssm_state, resid, norm_w=None, eps=0.0, normed=None):
        """xn [B, D] (model dtype).  Updates conv_state [B,Es,K-1] and
        ssm_state [B,Es,N] (fp32) in place; adds the output into resid."""
        self._check_states(conv_state, ssm_state)
        y = self._step_mix(self._in_proj(xn, "d_in_proj"), conv_state, ssm_state)
        partial_o = torch.empty(xn.shape[0], self.cfg.d_model, device=xn.device, dtype=torch.float32)
        self._gemm(y, self.out_proj.weight, partial_o, tag="d_out_proj")
        ev = _prof_begin()
        self._reduce_out(partial_o, resid, norm_w, eps, normed)
        _prof_end(ev, "d_reduce_out", 0)

    def _step_int8(self, rows, conv_state, ssm_state):
        """rows: int8 rows [B, D].  Updates the states in place; returns the mixer output fp32 [B, D]."""
        self._check_states(conv_state, ssm_state)
        return self._out_proj_int8(self._step_mix(self._in_proj(rows, "d_in_proj"), conv_state, ssm_state), "d_out_proj")

    def _check_states(self, conv_state, ssm_state):
        if ssm_state.dtype != torch.float32:
            raise TypeError("ssm_state must be float32 (allocate the cache with MambaCache.allocate)")
        if conv_state.dtype != self._dt():
            raise TypeError(f"conv_state dtype {conv_state.dtype} != model dtype {self._dt()}")

    def _step_mix(self, xz, conv_state, ssm_state):
        """From in_proj's output xz [B, 2Es] to out_proj's input y [B, Es]; the states are updated in place."""
        cfg = self.cfg
        es, n, r, k = self.es, cfg.d_state, cfg.dt_rank, cfg.d_conv
        Bn = xz.shape[0]
        dt_ = self._dt()
        dev = xz.device
        xc = torch.empty(Bn, es, device=dev, dtype=dt_)
        ev = _prof_begin()
        L.call("mtp_conv1d_silu", L.ptr(xz), 2 * es, L.ptr(self.conv1d.weight), L.ptr(self.conv1d.bias),
               L.ptr(conv_state), L.ptr(xc), es, Bn, 1, es, k, L.dtype_code(dt_), L.stream_ptr())
        _prof_end(ev, "d_conv", 0)
        partial_x = torch.empty(Bn, r + 2 * n, device=dev, dtype=torch.float32)
        self._gemm(xc, self.x_proj.weight, partial_x, tag="d_x_proj")
        dt_low = torch.empty(Bn, r, device=dev, dtype=dt_)
        bc = torch.empty(Bn, 2 * n, device=dev, dtype=torch.float32)
        ev = _prof_begin()
        self._reduce_x(partial_x, dt_low, bc)
        _prof_end(ev, "d_reduce_x", 0)
        y = torch.empty(Bn, es, device=dev, dtype=dt_)
        ev = _prof_begin()
        L.call("mtp_step", L.ptr(xz), 2 * es, L.ptr(dt_low), r, L.ptr(self.dt_proj.weight), L.ptr(self.dt_proj.bias),
               L.ptr(bc), 2 * n, L.ptr(self.A_log), L.ptr(self.D), L.ptr(self.conv1d.weight), L.ptr(self.conv1d.bias),
               L.ptr(conv_state), L.ptr(ssm_state), L.ptr(y), es, Bn, es, n, r, k, L.dtype_code(dt_), L.stream_ptr())
        _prof_end(ev, "d_step", 0)
        return y

    # ------------------------------------------------------------ reference-shaped API
    def prefill(self, x: torch.Tensor, cache=None):
        """x [b, l, d_model] -> (out [b, l, d_model], conv_state [b,Es,K-1], ssm_state [b,Es,N] fp32)
        (model.py:184-241 / tp_model.py:85-135).  The cache is read, not modified."""
        self._check_input(x, "prefill")
        b, l, d = x.shape
        xn = x.reshape(b * l, d).contiguous()
        ci = cache.conv_state if cache is not None and cache.conv_state is not None else None
        si = cache.ssm_state.float().contiguous() if cache is not None and cache.ssm_state is not None else None
        if self._int8 is not None:
            self._check_int8()
            out, cf, sf = self._prefill_int8(quantize_rows(xn), b, l, ci, si)
            return out.to(x.dtype).view(b, l, d), cf, sf
        resid = torch.zeros(b * l, d, device=x.device, dtype=torch.float32)
        cf, sf = self._prefill_core(xn, b, l, ci, si, resid)
        return resid.to(x.dtype).view(b, l, d), cf, sf

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        out, _, _ = self.prefill(x, cache=None)
        return out

    def step(self, x_t: torch.Tensor, cache):
        """x_t [b, d_model] -> out [b, d_model]; mutates the cache in place
        (model.py:249-294 / tp_model.py:137-179)."""
        self._check_input(x_t, "step")
        b, d = x_t.shape
        if self._int8 is not None:
            self._check_int8()
            return self._step_int8(quantize_rows(x_t), cache.conv_state, cache.ssm_state).to(x_t.dtype)
        resid = torch.zeros(b, d, device=x_t.device, dtype=torch.float32)
        self._step_core(x_t.contiguous(), cache.conv_state, cache.ssm_state, resid)
        return resid.to(x_t.dtype)
