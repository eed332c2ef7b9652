"""Two-layer MLP chain out = relu(relu(X @ W1 + b1) @ W2 + b2), each layer one fused call.

The direct consumer of the fused dense layer: layer 1 writes H into a caller-owned buffer,
layer 2 reads it; nothing else is materialised.  In BF16 mode the weights are rounded to
bf16 once (tforge_convert_bf16) and passed as bf16 operands, and H is kept in bf16 by
default: layer 1's epilogue rounds its output to bf16 (out_dtype = TFORGE_BF16), which is
exactly what layer 2 would do to an f32 H before its MMAs, so the result is the same bits
with half the H traffic and no conversion pass (`--h-dtype f32` keeps an f32 H).  Rows of X shard over GPUs like tensorforge_b200.shard: weights are
broadcast once, H and the output stay on the rank that owns the rows.

    python -m tensorforge_b200.mlp --shape 65536x4096x16384 --mode fp32        # one GPU
    torchrun --nproc-per-node 8 -m tensorforge_b200.mlp --shape 65536x4096x16384  # M-sharded

`FeedForward` is the transformer block around two layers -- residual, norm, activation, bf16 with its
gradient or 8-bit operands -- and `--block` times it:

    python -m tensorforge_b200.mlp --block --shape 8192x4096x16384 --mode bf16 --train
"""

from __future__ import annotations

import argparse
import json
import os
import sys

from . import _lib
from .shard import broadcast_weights, row_partition


class MLP2:
    """relu(relu(X @ W1 + b1) @ W2 + b2) on torch tensors of one GPU, through the C-ABI."""

    def __init__(self, w1, b1, w2, b2, mode: str = "fp32", h_bf16: bool | None = None):
        import torch

        self.mode = mode
        # BF16 mode: H in bf16 unless asked otherwise; other modes keep an f32 H.
        self.h_bf16 = (mode == "bf16") if h_bf16 is None else bool(h_bf16)
        if self.h_bf16 and mode != "bf16":
            raise ValueError("a bf16 H needs mode='bf16'")
        self.b1, self.b2 = b1, b2
        self.d, self.h = w1.shape
        if w2.shape != (self.h, self.d) or b1.shape != (self.h,) or b2.shape != (self.d,):
            raise ValueError("MLP2 expects W1 d x h, b1 h, W2 h x d, b2 d")
        if mode == "bf16":
            # Weights converted once; activations are converted inside each call.
            L = _lib.lib()
            self.w1 = torch.empty(w1.shape, device=w1.device, dtype=torch.bfloat16)
            self.w2 = torch.empty(w2.shape, device=w2.device, dtype=torch.bfloat16)
            stream = torch.cuda.current_stream(w1.device).cuda_stream
            _lib.check(L.tforge_convert_bf16(w1.data_ptr(), self.w1.data_ptr(), w1.numel(), stream), "convert W1")
            _lib.check(L.tforge_convert_bf16(w2.data_ptr(), self.w2.data_ptr(), w2.numel(), stream), "convert W2")
            self.b_dtype = _lib.BF16
        else:
            self.w1, self.w2 = w1, w2
            self.b_dtype = _lib.F32

    @property
    def h_dtype(self):
        import torch

        return torch.bfloat16 if self.h_bf16 else torch.float32

    def layer(self, x, w, b, out, stream) -> None:
        import torch

        m, k = x.shape
        n = w.shape[1]
        dt = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
        _lib.gemm("mbr", x.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, self.mode, bias=b.data_ptr(),
                  stream=stream, a_dtype=dt[x.dtype], b_dtype=self.b_dtype, out_dtype=dt[out.dtype])

    def __call__(self, x, h=None, out=None, stream=None):
        import torch

        m = x.shape[0]
        if h is None:
            h = torch.empty((m, self.h), device=x.device, dtype=self.h_dtype)
        if out is None:
            out = torch.empty((m, self.d), device=x.device, dtype=torch.float32)
        if stream is None:
            stream = torch.cuda.current_stream(x.device).cuda_stream
        self.layer(x, self.w1, self.b1, h, stream)
        self.layer(h, self.w2, self.b2, out, stream)
        return h, out


class FeedForward:
    """A transformer's feed-forward block on torch tensors of one GPU, through the C-ABI:

        s = x + residual;  out = s + act(rms_norm(s) @ W1 + b1) @ W2 + b2

    x, residual, s and out are bf16, M x D; W1 is D x H, W2 H x D.  mode "bf16": weights in bf16 as
    given.  mode "fp8": each output feature's weights in 8 bits with a scale, the activations in 8
    bits with a scale a row -- the norm writes the first product's, the quantizer the second's.
    bf16 weights and f32 vectors that are contiguous are used where they are, so that steps of an
    optimizer reach the block; others, and all weights in mode "fp8", are copied as they are now, on the
    current stream (a call on another one waits for it first, as for any tensor made there).
    autograd does not see the block: x and the residual may not need a gradient where autograd records
    (ValueError).
    x is on the weights' GPU, and calls run on its current stream.  `__call__(..., keep=True)` keeps what
    `backward` needs until it is called, on the same stream (mode "bf16"): x or s among it, which may
    not change before then.  `backward` gives it back, so the two are captured into a graph together or
    not at all."""

    def __init__(self, w1, b1, w2, b2, norm_weight, activation: str = "gelu_tanh", mode: str = "bf16", eps: float = 1e-5):
        import torch

        if mode not in ("bf16", "fp8"):
            raise ValueError("FeedForward takes mode 'bf16' or 'fp8'")
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        self.d, self.h = w1.shape
        if w2.shape != (self.h, self.d) or b1.shape != (self.h,) or b2.shape != (self.d,) or norm_weight.shape != (self.d,):
            raise ValueError("FeedForward expects W1 d x h, b1 h, W2 h x d, b2 d, norm weight d")
        if w1.device.type != "cuda" or any(t.device != w1.device for t in (b1, w2, b2, norm_weight)):
            raise ValueError("FeedForward expects its weights on one GPU")
        self.mode, self.activation, self.eps = mode, activation, eps
        w1, w2 = w1.detach(), w2.detach()
        self.b1, self.b2, self.norm_weight = (t.detach().float().contiguous() for t in (b1, b2, norm_weight))
        self.kept = None
        if mode == "bf16":
            self.w1, self.w2 = w1.bfloat16().contiguous(), w2.bfloat16().contiguous()
            return
        with torch.cuda.device(w1.device):
            self.w1, self.s1 = self._quantize(w1.float().t().contiguous())
            self.w2, self.s2 = self._quantize(w2.float().t().contiguous())

    @staticmethod
    def _stream(t):
        import torch

        return torch.cuda.current_stream(t.device).cuda_stream

    def _quantize(self, x):
        """Rows of x (f32 or bf16) in 8 bits, and their scales."""
        import torch

        m, n = x.shape
        q = torch.empty((m, n), device=x.device, dtype=torch.float8_e4m3fn)
        scale = torch.empty((m,), device=x.device)
        _lib.quantize_e4m3(x.data_ptr(), q.data_ptr(), scale.data_ptr(), m, n,
                           _lib.F32 if x.dtype == torch.float32 else _lib.BF16, stream=self._stream(x))
        return q, scale

    def __call__(self, x, residual=None, keep: bool = False):
        """(out, s).  s is what the next block adds its own output to when blocks are chained by hand;
        out already holds it."""
        import torch

        if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != self.d or not x.is_contiguous():
            raise ValueError("FeedForward takes contiguous bf16 rows of its width")
        if x.device != self.b1.device or (residual is not None and residual.device != x.device):
            raise ValueError("FeedForward takes rows on its weights' GPU")
        if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape or not residual.is_contiguous()):
            raise ValueError("the residual is like x")
        if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
            raise ValueError("FeedForward's gradients come from its backward(): detach its inputs")
        if keep and self.mode != "bf16":
            raise ValueError("only mode 'bf16' has a gradient")
        m, fp8 = x.shape[0], self.mode == "fp8"
        with torch.cuda.device(x.device):
            st = self._stream(x)
            capturing = keep and torch.cuda.is_current_stream_capturing()

            def new(*shape, dtype=torch.bfloat16):
                return torch.empty(shape, device=x.device, dtype=dtype)

            s = new(m, self.d) if residual is not None else x
            n = new(m, self.d, dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16)
            scale = new(m, dtype=torch.float32) if fp8 else None
            rstd = new(m, dtype=torch.float32) if keep else None
            _lib.rms_norm(x.data_ptr(), n.data_ptr(), m, self.d, self.eps, weight=self.norm_weight.data_ptr(),
                          residual=residual.data_ptr() if residual is not None else None,
                          sum_out=s.data_ptr() if residual is not None else None, rstd=rstd.data_ptr() if keep else None,
                          scale=scale.data_ptr() if fp8 else None, out_dtype=_lib.E4M3 if fp8 else _lib.BF16, stream=st)
            hid, out = new(m, self.h), new(m, self.d)
            pre = new(m, self.h) if keep and self.activation != "none" else None
            if fp8:
                e4m3 = dict(a_dtype=_lib.E4M3, b_dtype=_lib.E4M3, trans_b=True, stream=st)
                _lib.linear(n.data_ptr(), self.w1.data_ptr(), hid.data_ptr(), m, self.h, self.d, self.activation,
                            bias=self.b1.data_ptr(), a_scale=scale.data_ptr(), b_scale=self.s1.data_ptr(), **e4m3)
                q, qs = self._quantize(hid)
                _lib.linear(q.data_ptr(), self.w2.data_ptr(), out.data_ptr(), m, self.d, self.h, bias=self.b2.data_ptr(),
                            residual=s.data_ptr(), a_scale=qs.data_ptr(), b_scale=self.s2.data_ptr(), **e4m3)
            else:
                _lib.linear(n.data_ptr(), self.w1.data_ptr(), hid.data_ptr(), m, self.h, self.d, self.activation,
                            bias=self.b1.data_ptr(), pre=pre.data_ptr() if pre is not None else None, stream=st)
                _lib.linear(hid.data_ptr(), self.w2.data_ptr(), out.data_ptr(), m, self.d, self.h, bias=self.b2.data_ptr(),
                            residual=s.data_ptr(), stream=st)
        if keep:
            self.kept = (s, rstd, n, pre, hid, st, capturing)
        return out, s

    def backward(self, dout) -> dict:
        """Gradients from out's gradient (bf16, M x D): dx (the residual's too), dw1, db1, dw2, db2 and
        dnorm_weight; the weights' in bf16, the vectors' in f32."""
        import torch

        if self.kept is None:
            raise ValueError("backward needs a call with keep=True before it")
        s, rstd, n, pre, hid, st, capturing = self.kept
        if dout.dtype != torch.bfloat16 or dout.shape != s.shape or not dout.is_contiguous() or dout.device != s.device:
            raise ValueError("backward takes out's gradient: contiguous bf16 rows like out's")
        if self._stream(s) != st:
            raise ValueError("backward runs on the stream of the call that it follows")
        m = s.shape[0]
        with torch.cuda.device(s.device):
            if torch.cuda.is_current_stream_capturing() != capturing:
                raise ValueError("backward is captured together with the call that it follows, or neither is")
            self.kept = None

            def new(*shape, dtype=torch.bfloat16):
                return torch.empty(shape, device=s.device, dtype=dtype)

            g = {"dx": new(m, self.d), "dw1": new(self.d, self.h), "db1": new(self.h, dtype=torch.float32),
                 "dw2": new(self.h, self.d), "db2": new(self.d, dtype=torch.float32),
                 "dnorm_weight": new(self.d, dtype=torch.float32)}
            dhid, dn = new(m, self.h), new(m, self.d)
            _lib.linear_backward(dout.data_ptr(), hid.data_ptr(), self.w2.data_ptr(), m, self.d, self.h, dA=dhid.data_ptr(),
                                 dB=g["dw2"].data_ptr(), dbias=g["db2"].data_ptr(), stream=st)
            _lib.linear_backward(dhid.data_ptr(), n.data_ptr(), self.w1.data_ptr(), m, self.h, self.d, self.activation,
                                 pre=pre.data_ptr() if pre is not None else None, dA=dn.data_ptr(), dB=g["dw1"].data_ptr(),
                                 dbias=g["db1"].data_ptr(), stream=st)
            _lib.rms_norm_backward(dn.data_ptr(), s.data_ptr(), rstd.data_ptr(), g["dx"].data_ptr(), m, self.d,
                                   weight=self.norm_weight.data_ptr(), ds=dout.data_ptr(), dweight=g["dnorm_weight"].data_ptr(),
                                   stream=st)
        return g


def flops(m: int, d: int, h: int) -> float:
    """2 M N K per layer (the reference's convention), two layers."""
    return 2.0 * m * d * h * 2


def block_errors(model, x, residual, out, rows, dout=None, grads=None, units=None, chunk: int = 1024) -> dict:
    """Relative errors (of norms) of a FeedForward block's output in `rows` and, with `grads`, of its
    gradients, against 64 bits from the block's own 8- or 16-bit weights (tanh gelu): dx in `rows`,
    what belongs to the hidden `units` of dw1, db1 and dw2, all of db2, and the norm weight's in as
    many columns, for which every row goes through both products, `chunk` at a time."""
    import math

    import torch

    if model.mode == "fp8":
        w1, w2 = (model.w1.double() * model.s1.double()[:, None]).t(), (model.w2.double() * model.s2.double()[:, None]).t()
    else:
        w1, w2 = model.w1.double(), model.w2.double()
    weight, b1, b2 = model.norm_weight.double(), model.b1.double(), model.b2.double()
    c = math.sqrt(2 / math.pi)

    def forward(at):
        s = x[at].double() + (residual[at].double() if residual is not None else 0.0)
        rstd = (s.square().mean(1, keepdim=True) + model.eps).rsqrt()
        return s, rstd, s * rstd * weight

    def act(z):
        """The activation and its slope."""
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)

    def error(got, want):
        return float((got.double() - want).norm() / want.norm())

    s, rstd, n = forward(rows)
    hid, slope = act(n @ w1 + b1)
    errors = {"out": error(out[rows], s + hid @ w2 + b2)}
    if grads is None:
        return errors
    d = dout[rows].double()
    dn = (d @ w2.t() * slope) @ w1.t()
    g, h = dn * weight, s * rstd
    errors["dx"] = error(grads["dx"][rows], rstd * (g - h * (g * h).mean(1, keepdim=True)) + d)
    cols = units % x.shape[1]
    dw1, dw2 = torch.zeros_like(w1[:, units]), torch.zeros_like(w2[units])
    db1, db2, dweight = torch.zeros_like(b1[units]), torch.zeros_like(b2), torch.zeros_like(weight[cols])
    for r0 in range(0, x.shape[0], chunk):
        at = slice(r0, r0 + chunk)
        s, rstd, n = forward(at)
        d = dout[at].double()
        hid, slope = act(n @ w1 + b1)
        dz = d @ w2.t() * slope
        dw1 += n.t() @ dz[:, units]
        db1 += dz[:, units].sum(0)
        dw2 += hid[:, units].t() @ d
        db2 += d.sum(0)
        dweight += (dz @ w1[cols].t() * (s * rstd)[:, cols]).sum(0)
    for name, got, want in (("dw1", grads["dw1"][:, units], dw1), ("db1", grads["db1"][units], db1), ("dw2", grads["dw2"][units], dw2),
                            ("db2", grads["db2"], db2), ("dnorm_weight", grads["dnorm_weight"][cols], dweight)):
        errors[name] = error(got, want)
    return errors


def block_bound(mode: str, name: str) -> float:
    """How far block_errors may be.  Of the output, the whole row's: two roundings of the activations (2^-8
    each way, or 2^-4 in 8 bits) and one of the output; of a gradient at most six values on the way in
    bf16 (n, pre, hid, dhid, dz, dn), half a step each."""
    if name != "out":
        return 6 * 2.0 ** -8
    return 2.0 ** -3 if mode == "fp8" else 2.0 ** -6


def run_block(args, x, w1, b1, w2, b2, world: int, rank: int) -> int:
    """Times the FeedForward block (with --train and its gradient) on this rank's rows and checks a
    seeded subset of its outputs and gradients against 64 bits."""
    import numpy as np
    import torch
    import torch.distributed as dist

    dev = x.device
    g = torch.Generator(device=dev)
    g.manual_seed(9)  # the same norm weight on every rank
    norm_weight = 1 + 0.2 * torch.randn(args.d, device=dev, generator=g)
    model = FeedForward(w1, b1, w2, b2, norm_weight, mode=args.mode)
    x = x.bfloat16()
    g.manual_seed(200 + rank)
    residual = torch.randn(x.shape, device=dev, generator=g).bfloat16()
    dout = (0.01 * torch.randn(x.shape, device=dev, generator=g)).bfloat16()

    def step():
        out, _ = model(x, residual, keep=args.train)
        return out, model.backward(dout) if args.train else None

    for _ in range(args.warmup):
        step()
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream(dev)
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    if world > 1:
        dist.barrier()
    e0.record(stream)
    for _ in range(args.steps):
        out, grads = step()
    e1.record(stream)
    torch.cuda.synchronize()
    ms = torch.tensor([e0.elapsed_time(e1) / args.steps], device=dev, dtype=torch.float64)
    if world > 1:
        dist.all_reduce(ms, op=dist.ReduceOp.MAX)
    status = _lib.device_status(stream.cuda_stream)

    rng = np.random.default_rng(rank)
    pick = lambda n: torch.from_numpy(np.sort(rng.choice(n, min(args.check_rows, n), replace=False))).to(dev)  # noqa: E731
    sel = pick(x.shape[0])
    errors = block_errors(model, x, residual, out, sel, dout, grads, pick(args.h)) if len(sel) else {"out": 0.0}
    # (A NaN is not within its bound.)
    ok = torch.tensor([int(status == 0 and all(e <= block_bound(args.mode, name) for name, e in errors.items()))], device=dev)
    if world > 1:
        dist.all_reduce(ok, op=dist.ReduceOp.MIN)
    if rank == 0:
        t = float(ms.item())
        fl = flops(args.m, args.d, args.h) * (3 if args.train else 1)
        line = {"workload": f"feed-forward block X {args.m}x{args.d}, W1 {args.d}x{args.h}, W2 {args.h}x{args.d}",
                "mode": args.mode, "gradient": bool(args.train), "n_gpus": world, "ms_per_step": t,
                "tflops": fl / (t * 1e-3) / 1e12, "rel_err": errors["out"], "rel_err_bound": block_bound(args.mode, "out"),
                "checked_rows_per_rank": int(len(sel)), "pass": bool(ok.item())}
        if args.train:
            line["gradient_rel_err"] = {k: e for k, e in errors.items() if k != "out"}
            line["gradient_rel_err_bound"] = block_bound(args.mode, "dx")
        print(json.dumps(line), flush=True)
    return 0 if ok.item() else 1


def main(argv=None) -> int:
    import numpy as np
    import torch
    import torch.distributed as dist

    from . import tforge_cpu as tc

    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--shape", default="65536x4096x16384",
                    help="MxDxH: rows of X in total (sharded over ranks), model width, hidden width")
    ap.add_argument("--mode", default="fp32", choices=["fp32", "tf32", "bf16", "fp8"])
    ap.add_argument("--block", action="store_true",
                    help="the transformer block around the two layers (norm, residual, gelu; bf16 or fp8)")
    ap.add_argument("--train", action="store_true", help="with --block: time the gradient too (bf16)")
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--check-rows", type=int, default=16, help="rows checked against FP64 per layer")
    ap.add_argument("--h-dtype", default="auto", choices=["auto", "f32", "bf16"],
                    help="hidden activation storage (auto: bf16 in BF16 mode, else f32)")
    args = ap.parse_args(argv)
    args.m, args.d, args.h = (int(x) for x in args.shape.lower().split("x"))
    if args.block != (args.mode == "fp8") and not (args.block and args.mode == "bf16"):
        ap.error("--block takes --mode bf16 or fp8, and fp8 needs --block")
    if args.train and not (args.block and args.mode == "bf16"):
        ap.error("--train needs --block --mode bf16")

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    if world > 1:
        import datetime

        dist.init_process_group("nccl", device_id=dev, timeout=datetime.timedelta(seconds=120))
    r0, r1 = row_partition(args.m, world, rank)
    rows = r1 - r0
    # Xavier-uniform weights, N(0, 0.02) biases, X U[-1, 1]; X rows generated per rank.
    g = torch.Generator(device=dev)
    g.manual_seed(100 + rank)
    x = torch.empty((rows, args.d), device=dev).uniform_(-1, 1, generator=g)
    lim = float(np.sqrt(6.0 / (args.d + args.h)))
    w1 = torch.empty((args.d, args.h), device=dev)
    w2 = torch.empty((args.h, args.d), device=dev)
    b1 = torch.empty((args.h,), device=dev)
    b2 = torch.empty((args.d,), device=dev)
    if rank == 0:
        g0 = torch.Generator(device=dev)
        g0.manual_seed(5)
        w1.uniform_(-lim, lim, generator=g0)
        w2.uniform_(-lim, lim, generator=g0)
        b1.normal_(0.0, 0.02, generator=g0)
        b2.normal_(0.0, 0.02, generator=g0)
    broadcast_weights(w1, b1)
    broadcast_weights(w2, b2)
    if args.block:
        rc = run_block(args, x, w1, b1, w2, b2, world, rank)
        if world > 1:
            dist.barrier()
            dist.destroy_process_group()
        return rc
    model = MLP2(w1, b1, w2, b2, args.mode, None if args.h_dtype == "auto" else args.h_dtype == "bf16")
    h = torch.empty((rows, args.h), device=dev, dtype=model.h_dtype)
    out = torch.empty((rows, args.d), device=dev)
    stream = torch.cuda.current_stream(dev)
    for _ in range(args.warmup):
        model(x, h, out)
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    if world > 1:
        dist.barrier()
    e0.record(stream)
    for _ in range(args.steps):
        model(x, h, out)
    e1.record(stream)
    torch.cuda.synchronize()
    ms = torch.tensor([e0.elapsed_time(e1) / args.steps], device=dev, dtype=torch.float64)
    if world > 1:
        dist.all_reduce(ms, op=dist.ReduceOp.MAX)
    status = _lib.device_status(stream.cuda_stream)

    # Per-layer FP64 check on a seeded subset of this rank's rows (layer 2 on our own H).
    sel = np.sort(np.random.default_rng(rank).choice(rows, min(args.check_rows, rows), replace=False))
    xs, hs, os_ = x[sel].cpu().numpy(), h[sel].float().cpu().numpy(), out[sel].cpu().numpy()
    r_1 = tc.check_output("mbr", {"a": xs, "b": w1.cpu().numpy(), "bias": b1.cpu().numpy()}, hs, args.mode,
                          out_unit=2.0 ** -8 if model.h_bf16 else 0.0)
    r_2 = tc.check_output("mbr", {"a": hs, "b": w2.cpu().numpy(), "bias": b2.cpu().numpy()}, os_, args.mode)
    ok = torch.tensor([int(r_1["pass"] and r_2["pass"] and status == 0)], device=dev)
    if world > 1:
        dist.all_reduce(ok, op=dist.ReduceOp.MIN)
    if rank == 0:
        t = float(ms.item())
        print(json.dumps({"workload": f"mlp2 X {args.m}x{args.d}, W1 {args.d}x{args.h}, W2 {args.h}x{args.d}",
                          "mode": args.mode, "h_dtype": "bf16" if model.h_bf16 else "f32",
                          "n_gpus": world, "ms_per_step": t,
                          "tflops": flops(args.m, args.d, args.h) / (t * 1e-3) / 1e12,
                          "err_over_bound_layer1": r_1["err_over_bound"], "err_over_bound_layer2": r_2["err_over_bound"],
                          "checked_rows_per_rank": int(len(sel)), "pass": bool(ok.item())}), flush=True)
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()
    return 0 if ok.item() else 1


if __name__ == "__main__":
    sys.exit(main())
