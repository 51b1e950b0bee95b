"""The operators around a selective state space layer, as cases that can be timed: the short causal convolution, the
selective scan with a decay per channel and state column, the root-mean-square norm with the residual's addition, each
for prompts, for training and for generation steps.

``kind`` of a case says which operator it calls:

  "conv"        short_conv on a batch or on packed sequences; with ``train`` its gradients as well
  "conv_step"   short_conv_step: one token of each sequence, the convolution's state goes from one cache to another
  "scan"        selective_scan on a batch or on packed sequences; with ``train`` its gradients as well
  "scan_step"   selective_scan_step: one token of each sequence
  "norm"        rms_norm with the residual's addition and all gradients
  "norm_quant"  rms_norm_quant: the same norm with an output in 8 bits and its scales

With ``own`` false every operator is computed in its plain form, elementary torch operations in 32 bits.
"""
import os
import sys

import torch

own = False  # whether run() calls the package's operators

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _package():
    path = os.path.join(os.getcwd(), "mamba-ascendc_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    import ascend_kernel

    return ascend_kernel


# ---------------------------------------------------------------------------------------------------- the cases
def _conv(name, batch, length, channels, width, dtype, packed=0, train=False, sliced=False, start=True):
    case = dict(kind="conv", batch=batch, length=length, channels=channels, width=width, dtype=dtype, packed=packed,
                train=train, sliced=sliced, start=start)
    return dict(name=name, **case) if name else case


def _conv_step(name, batch, channels, width, dtype, slots):
    case = dict(kind="conv_step", batch=batch, channels=channels, width=width, dtype=dtype, slots=slots)
    return dict(name=name, **case) if name else case


def _scan(name, batch, length, channels, state, groups, dtype, packed=0, train=False, start=False):
    case = dict(kind="scan", batch=batch, length=length, channels=channels, state=state, groups=groups, dtype=dtype,
                packed=packed, train=train, start=start)
    return dict(name=name, **case) if name else case


def _scan_step(name, batch, channels, state, groups, dtype, slots):
    case = dict(kind="scan_step", batch=batch, channels=channels, state=state, groups=groups, dtype=dtype, slots=slots)
    return dict(name=name, **case) if name else case


def _norm(name, rows, width, dtype):
    case = dict(kind="norm", rows=rows, width=width, dtype=dtype)
    return dict(name=name, **case) if name else case


def _norm_quant(name, rows, width, dtype, group):
    case = dict(kind="norm_quant", rows=rows, width=width, dtype=dtype, group=group)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one generation step of 16 sequences through a layer of 24 heads of 64 with two states of 128: 1792 channels
        _conv_step("conv_step_16", 16, 1792, 4, "fp32", slots=False),
        # a generation step of a full serving batch, the states in a cache of slots, the batch padded
        _conv_step("conv_step_slots", 256, 8192, 4, "bf16", slots=True),
        # eleven prompts of odd lengths packed one behind another, each with its own state
        _conv("conv_prompts", 1, 8191, 4096, 4, "bf16", packed=11),
        # the convolution of a Vision-Mamba2 block in training: 4 images, a column slice of the input projection
        _conv("conv_train_vision", 4, 4096, 512, 4, "fp32", train=True, sliced=True, start=False),
        # the smallest step of the recurrence: one sequence, launch and host work count
        _scan_step("scan_step_1", 1, 1536, 16, 1, "bf16", slots=False),
        # a generation step of a full serving batch from a cache of slots: reading and writing the states
        _scan_step("scan_step_slots", 256, 4096, 16, 1, "bf16", slots=True),
        # prefill of one long prompt
        _scan("scan_prompt", 1, 8192, 4096, 16, 1, "bf16"),
        # a training step of the recurrence, ragged length
        _scan("scan_train", 4, 2000, 2048, 16, 1, "bf16", train=True),
        # the norm in front of a Vision-Mamba2 block in training: 4 images of 4096 tokens, width 192
        _norm("norm_train_vision", 16384, 192, "fp32"),
        # the norm of a wide layer in training
        _norm("norm_train_wide", 8192, 4096, "bf16"),
        # a generation step of 16 sequences in front of a projection in 8 bits, one scale per token
        _norm_quant("norm_quant_16", 16, 4096, "bf16", 0),
        # a long prompt, one scale per 128 columns
        _norm_quant("norm_quant_prompt", 16384, 4096, "bf16", 128),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step", "norm", "norm_quant"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    channels = _log_int(rng, 64, 8192)
    if rng.random() < 0.7:
        channels = max(64, channels // 64 * 64)
    if kind == "conv_step":
        return _conv_step(None, _log_int(rng, 1, 256), channels, rng.choice([2, 3, 4, 4]), dtype, rng.random() < 0.5)
    if kind == "norm":
        return _norm(None, min(_log_int(rng, 1, 65536), 8192 * 4096 // channels), channels, dtype)
    if kind == "norm_quant":
        channels = max(128, channels // 128 * 128)
        return _norm_quant(None, min(_log_int(rng, 1, 65536), 16384 * 4096 // channels), channels, dtype,
                           rng.choice([0, 0, 64, 128]))
    packed = rng.choice([0, 0, _log_int(rng, 1, 40)])
    train = not packed and rng.random() < 0.5
    batch = 1 if packed else _log_int(rng, 1, 8)
    length = _log_int(rng, 1, 16384)
    if kind == "conv":
        length = max(1, min(length, 8191 * 4096 // (batch * channels)))
        return _conv(None, batch, length, channels, rng.choice([2, 3, 4, 4]), dtype, packed, train, rng.random() < 0.4,
                     rng.random() < 0.5)
    groups = rng.choice([1, 1, 2, 4])
    channels = max(64, min(channels, 4096)) // groups * groups
    state = rng.choice([16, 16, 16, 8, 24, 64])
    if kind == "scan_step":
        return _scan_step(None, min(_log_int(rng, 1, 256), 256 * 16 // state), channels, state, groups, dtype,
                          rng.random() < 0.5)
    most = 4 * 2000 * 2048 * 16 if train else 8192 * 4096 * 16
    length = max(1, min(length, most // (batch * channels * state)))
    return _scan(None, batch, length, channels, state, groups, dtype, packed, train, rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------- inputs
def _lengths(total, count, gen):
    """`count` lengths that add up to `total`, some of them one or none."""
    cuts = sorted(int(total * f) for f in torch.rand(count - 1, generator=gen).tolist())
    edges = [0] + cuts + [total]
    return [b - a for a, b in zip(edges[:-1], edges[1:])]


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], _TYPES[case["dtype"]]

    def normal(*shape, type_=dtype, scale=1.0, shift=0.0):
        return (shift + scale * torch.randn(*shape, generator=gen, device="cuda")).to(type_)

    f32 = torch.float32
    s = {"case": case}
    if kind in ("norm", "norm_quant"):
        rows, width = case["rows"], case["width"]
        # the residual stream is some times larger than what a layer adds to it, and some of its columns stand out
        s["x"], s["weight"] = normal(rows, width), normal(width, type_=f32, scale=0.1, shift=1.0)
        s["residual"] = (torch.randn(rows, width, generator=gen, device="cuda") *
                         (1 + 8 * torch.rand(width, generator=gen, device="cuda") ** 8)).to(dtype)
        if kind == "norm":
            s["dout"], s["dresidual"] = normal(rows, width), normal(rows, width)
            s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "weight", "residual")]
        return s

    channels = case["channels"]
    batch = case["batch"]
    step = kind in ("conv_step", "scan_step")
    lengths = None
    if not step:
        tokens = case["length"]
        if case["packed"]:
            lengths = _lengths(tokens, case["packed"], host)
            edges = [0]
            for n in lengths:
                edges.append(edges[-1] + n)
            s["cu_seqlens"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
        s["lengths"] = lengths
    rows = case["packed"] if not step and case["packed"] else batch
    if step and case["slots"]:
        pool = batch + batch // 4 + 1
        slots = torch.randperm(pool, generator=host)[:batch].to(torch.int32)
        slots[batch - batch // 16:] = -1  # the batch is padded to its size
        s["slots"] = slots.cuda()
    elif step:
        pool, s["slots"] = batch, None
    lead = (batch,) if step else (batch, tokens)
    if kind in ("conv", "conv_step"):
        width = case["width"]
        if kind == "conv" and case["sliced"]:
            extra = 96
            s["x"] = normal(*lead, channels + extra)[..., 64:64 + channels]
        else:
            s["x"] = normal(*lead, channels)
        s["weight"] = normal(channels, width, type_=f32, scale=width ** -0.5)
        s["bias"] = normal(channels, type_=f32, scale=0.1)
        if step:
            s["state"] = normal(pool, width - 1, channels)
            s["state_out"] = torch.zeros_like(s["state"])
            return s
        s["initial"] = normal(rows, width - 1, channels) if case["start"] else None
        if case["train"]:
            s["dout"], s["dfinal"] = normal(*lead, channels), normal(rows, width - 1, channels)
            s["leaves"] = [t.detach().requires_grad_(True) for t in (s["x"], s["weight"], s["bias"], s["initial"])
                           if t is not None]
            s["x"], s["weight"], s["bias"] = s["leaves"][:3]
            if s["initial"] is not None:
                s["initial"] = s["leaves"][3]
        return s

    state, groups = case["state"], case["groups"]
    s["x"], s["z"] = normal(*lead, channels), normal(*lead, channels)
    s["dt"] = normal(*lead, channels, scale=0.5)
    s["B"], s["C"] = normal(*lead, groups, state), normal(*lead, groups, state)
    # decays as a trained layer has them: about 1 to `state` per channel, steps of 0.001 to 0.1
    s["A"] = -(torch.arange(1, state + 1, device="cuda") * torch.exp(normal(channels, state, type_=f32, scale=0.1)))
    steps = 10 ** (-3 + 2 * torch.rand(channels, generator=gen, device="cuda"))
    s["dt_bias"] = steps + torch.log(-torch.expm1(-steps))
    s["D"] = normal(channels, type_=f32, scale=0.1, shift=1.0)
    if step:
        s["state"] = normal(pool, channels, state, type_=f32)
        s["state_out"] = torch.zeros_like(s["state"])
        return s
    s["initial"] = normal(rows, channels, state, type_=f32) if case["start"] else None
    if case["train"]:
        s["dout"], s["dfinal"] = normal(*lead, channels), normal(rows, channels, state, type_=f32, scale=0.1)
        s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial")
                       if s[k] is not None]
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    return (_run_own if own else _run_plain)[kind](state)


def _own_conv(s):
    ak, case = _package(), s["case"]
    if not case["train"]:
        with torch.no_grad():
            return list(ak.short_conv(s["x"], s["weight"], s["bias"], activation="silu", initial_states=s["initial"],
                                      cu_seqlens=s.get("cu_seqlens"), return_final_state=True))
    out, final = ak.short_conv(s["x"], s["weight"], s["bias"], activation="silu", initial_states=s["initial"],
                               return_final_state=True)
    grads = torch.autograd.grad([out, final], s["leaves"], [s["dout"], s["dfinal"]])
    return [out.detach(), final.detach(), *grads]


def _own_conv_step(s):
    with torch.no_grad():
        out = _package().short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu", slots=s["slots"],
                                         state_out=s["state_out"])
    return [out, s["state_out"]]


def _own_scan(s):
    ak, case = _package(), s["case"]
    arguments = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True, initial_states=s["initial"],
                     return_final_state=True)
    if not case["train"]:
        with torch.no_grad():
            return list(ak.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], cu_seqlens=s.get("cu_seqlens"),
                                          **arguments))
    out, final = ak.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], **arguments)
    grads = torch.autograd.grad([out, final], s["leaves"], [s["dout"], s["dfinal"]])
    return [out.detach(), final.detach(), *grads]


def _own_scan_step(s):
    with torch.no_grad():
        out = _package().selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                             dt_bias=s["dt_bias"], dt_softplus=True, slots=s["slots"],
                                             state_out=s["state_out"])
    return [out, s["state_out"]]


def _own_norm(s):
    out, stream = _package().rms_norm(s["x"], s["weight"], residual=s["residual"], eps=1e-5)
    grads = torch.autograd.grad([out, stream], s["leaves"], [s["dout"], s["dresidual"]])
    return [out.detach(), stream.detach(), *grads]


def _own_norm_quant(s):
    return list(_package().rms_norm_quant(s["x"], s["weight"], residual=s["residual"], eps=1e-5,
                                          group_size=s["case"]["group"] or None))


# -- plain forms: batches of sequences [S, L, ...]; packed ones are laid out as such a batch and gathered again
def _unpack(s, t):
    """Packed [1, T, ...] as [S, longest, ...], zeros behind the end of each."""
    lengths = s["lengths"]
    if lengths is None:
        return t
    return torch.nn.utils.rnn.pad_sequence(list(torch.split(t[0], lengths)), batch_first=True)


def _pack(s, t):
    lengths = s["lengths"]
    if lengths is None:
        return t
    return torch.cat([t[i, :n] for i, n in enumerate(lengths)])[None]


def _plain_conv(s):
    case = s["case"]
    width, dtype = case["width"], s["x"].dtype
    with torch.no_grad():
        x = _unpack(s, s["x"]).float()
        rows, tokens, channels = x.shape
        w, bias = s["weight"].float(), s["bias"].float()
        start = x.new_zeros(rows, width - 1, channels) if s["initial"] is None else s["initial"].float()
        held = torch.cat([start, x], 1)  # token t stands at t + width - 1
        pre = bias + sum(held[:, k:k + tokens] * w[:, k] for k in range(width))
        gate = torch.sigmoid(pre)
        out = pre * gate
        if s["lengths"] is None:
            final = held[:, tokens:]
        else:
            final = torch.stack([held[i, n:n + width - 1] for i, n in enumerate(s["lengths"])])
        outputs = [_pack(s, out).to(dtype), final.to(dtype)]
        if not case["train"]:
            return outputs
        dpre = s["dout"].float() * (gate * (1 + pre * (1 - gate)))
        dheld = torch.zeros_like(held)
        for k in range(width):
            dheld[:, k:k + tokens] += dpre * w[:, k]
        dheld[:, tokens:] += s["dfinal"].float()
        dw = torch.stack([(dpre * held[:, k:k + tokens]).sum((0, 1)) for k in range(width)], 1)
        grads = [dheld[:, width - 1:].to(dtype), dw.to(s["weight"].dtype), dpre.sum((0, 1)).to(s["bias"].dtype)]
        if s["initial"] is not None:
            grads.append(dheld[:, :width - 1].to(dtype))
        return outputs + grads


def _plain_conv_step(s):
    width = s["case"]["width"]
    x, slots, dtype = s["x"], s["slots"], s["x"].dtype
    live = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if slots is None else slots >= 0
    at = torch.arange(x.shape[0], device=x.device) if slots is None else slots.clamp(min=0).long()
    held = torch.cat([s["state"][at], x[:, None]], 1)
    pre = s["bias"].float() + (held.float() * s["weight"].float().t()).sum(1)
    out = torch.where(live[:, None], pre * torch.sigmoid(pre), torch.zeros_like(pre)).to(dtype)
    s["state_out"][at[live]] = held[live, 1:]
    return [out, s["state_out"]]


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _prefix(a, b, flip=False):
    """h[t] = a[t] h[t-1] + b[t] from zero along dimension 1 (backwards with ``flip``: h[t] = a[t] h[t+1] + b[t]), and the
    products of the a, by doubling the distance."""
    n, step = a.shape[1], 1
    while step < n:
        if flip:
            b = torch.cat([b[:, :-step] + a[:, :-step] * b[:, step:], b[:, -step:]], 1)
            a = torch.cat([a[:, :-step] * a[:, step:], a[:, -step:]], 1)
        else:
            b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
            a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return a, b


_CHUNK = 64


def _heads(t, channels):
    """[S, L, G, N] as [S, L, C, N]."""
    groups = t.shape[-2]
    return t.float().repeat_interleave(channels // groups, dim=-2)


def _plain_scan(s):
    case = s["case"]
    with torch.no_grad():
        dtype = s["x"].dtype
        x, raw, z = (_unpack(s, s[k]).float() for k in ("x", "dt", "z"))
        bm, cm = (_unpack(s, s[k]) for k in ("B", "C"))
        rows, tokens, channels = x.shape
        A, D = s["A"].float(), s["D"].float()
        pre = raw + s["dt_bias"].float()
        dt = _softplus(pre)
        if s["lengths"] is not None:  # behind the end of a sequence its state stays
            ends = torch.tensor(s["lengths"], device=x.device)
            dt = dt * (torch.arange(tokens, device=x.device) < ends[:, None])[..., None]
        h = x.new_zeros(rows, channels, case["state"]) if s["initial"] is None else s["initial"].float()
        y = torch.empty_like(x)
        starts = []
        for t in range(0, tokens, _CHUNK):
            c = slice(t, min(tokens, t + _CHUNK))
            starts.append(h)
            a = torch.exp(dt[:, c, :, None] * A)
            products, local = _prefix(a, (dt[:, c] * x[:, c])[..., None] * _heads(bm[:, c], channels))
            states = local + products * h[:, None]
            y[:, c] = (states * _heads(cm[:, c], channels)).sum(-1)
            h = states[:, -1]
        skip = y + D * x
        gate = torch.sigmoid(z)
        outputs = [_pack(s, skip * z * gate).to(dtype), h]
        if not case["train"]:
            return outputs
        dout = s["dout"].float()
        dy = dout * z * gate
        dz = dout * skip * gate * (1 + z * (1 - gate))
        dx, ddt = dy * D, torch.empty_like(dt)
        dB, dC = torch.empty_like(bm, dtype=torch.float32), torch.empty_like(cm, dtype=torch.float32)
        dA = torch.zeros_like(A)
        g = s["dfinal"].float()  # gradient of the state behind the chunk
        groups = bm.shape[2]
        for k in reversed(range(len(starts))):
            c = slice(k * _CHUNK, min(tokens, (k + 1) * _CHUNK))
            h = starts[k]
            B, C = _heads(bm[:, c], channels), _heads(cm[:, c], channels)
            a = torch.exp(dt[:, c, :, None] * A)
            products, local = _prefix(a, (dt[:, c] * x[:, c])[..., None] * B)
            states = local + products * h[:, None]
            after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)  # decay on the way to the next token
            products, local = _prefix(after, dy[:, c, :, None] * C, flip=True)
            gt = local + products * g[:, None]
            g = a[:, 0] * gt[:, 0]
            before = torch.cat([h[:, None], states[:, :-1]], 1)
            dlog = gt * a * before  # gradient of dt * A
            through = (gt * B).sum(-1)
            dx[:, c] += dt[:, c] * through
            ddt[:, c] = (dlog * A).sum(-1) + x[:, c] * through
            dA += (dlog * dt[:, c, :, None]).sum((0, 1))
            fold = lambda v: v.unflatten(2, (groups, channels // groups)).sum(3)  # noqa: E731
            dB[:, c] = fold(gt * (dt[:, c] * x[:, c])[..., None])
            dC[:, c] = fold(states * dy[:, c, :, None])
        dpre = ddt * torch.sigmoid(pre)
        grads = [dx.to(dtype), dpre.to(dtype), dA, dB.to(dtype), dC.to(dtype), (dy * x).sum((0, 1)), dz.to(dtype),
                 dpre.sum((0, 1))]
        if s["initial"] is not None:
            grads.append(g)
        return outputs + grads


def _plain_scan_step(s):
    x, slots = s["x"].float(), s["slots"]
    channels = x.shape[1]
    live = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if slots is None else slots >= 0
    at = torch.arange(x.shape[0], device=x.device) if slots is None else slots.clamp(min=0).long()
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    h = s["state"][at] * torch.exp(dt[..., None] * s["A"]) + (dt * x)[..., None] * _heads(s["B"], channels)
    z = s["z"].float()
    out = ((h * _heads(s["C"], channels)).sum(-1) + s["D"] * x) * z * torch.sigmoid(z)
    s["state_out"][at[live]] = h[live]
    return [torch.where(live[:, None], out, torch.zeros_like(out)).to(s["x"].dtype), s["state_out"]]


def _plain_norm(s):
    with torch.no_grad():
        dtype, w = s["x"].dtype, s["weight"].float()
        v = s["x"].float() + s["residual"].float()
        r = torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5)
        unit = v * r
        dout = s["dout"].float()
        g = dout * w
        dv = r * (g - unit * (g * unit).mean(-1, keepdim=True)) + s["dresidual"].float()
        return [(unit * w).to(dtype), v.to(dtype), dv.to(dtype), (dout * unit).sum(0), dv.to(dtype)]


def _plain_norm_quant(s):
    v = s["x"].float() + s["residual"].float()
    rows, width = v.shape
    group = s["case"]["group"] or width
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
    y = y.view(rows, width // group, group)
    scale = y.abs().amax(-1) / 448
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (y / scale[..., None]).clamp(-448, 448).view(rows, width)
    return [q.to(torch.float8_e4m3fn), scale, v.to(s["x"].dtype)]


_run_plain = {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
              "norm": _plain_norm, "norm_quant": _plain_norm_quant}
_run_own = {"conv": _own_conv, "conv_step": _own_conv_step, "scan": _own_scan, "scan_step": _own_scan_step,
            "norm": _own_norm, "norm_quant": _own_norm_quant}


# ---------------------------------------------------------------------------------------------------- bytes and flops
def work(case):
    """Each input once and each output once; a multiplication with an addition counts two, an exponential one."""
    kind, e = case["kind"], _BYTES[case["dtype"]]
    if kind == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": float(n * e * 8 + 8 * case["width"]), "flops": 14.0 * n}
    if kind == "norm_quant":
        n = case["rows"] * case["width"]
        return {"bytes": float(n * (3 * e + 1) + 4 * n // (case["group"] or case["width"])), "flops": 7.0 * n}
    step = kind in ("conv_step", "scan_step")
    live = case["batch"] - (case["batch"] // 16 if step and case["slots"] else 0)
    tokens = live if step else case["batch"] * case["length"]
    rows = live if step else case["packed"] or case["batch"]
    n = tokens * case["channels"]
    if kind in ("conv", "conv_step"):
        width = case["width"]
        held = rows * (width - 1) * case["channels"] * e
        start = step or case["start"]
        moved = 2 * n * e + held * (2 if start else 1) + 4 * case["channels"] * (width + 1)
        flops = n * (2 * width + 4)
        if not step and case["train"]:
            moved += 3 * n * e + held * (3 if start else 1) + 8 * case["channels"] * (width + 1)
            flops += n * (6 * width + 8)
        return {"bytes": float(moved), "flops": float(flops)}
    state, groups = case["state"], case["groups"]
    held = rows * case["channels"] * state * 4
    start = step or case["start"]
    shared = 2 * tokens * groups * state * e
    weights = 4 * case["channels"] * (state + 2)
    moved = 4 * n * e + shared + weights + held * (2 if start else 1)
    flops = n * (7 * state + 10)
    if not step and case["train"]:
        moved += 7 * n * e + 2 * shared + 2 * weights + held * (3 if start else 1)
        flops += n * (22 * state + 20)
    return {"bytes": float(moved), "flops": float(flops)}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions token by token in 64 bits."""
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in prepare(case, seed).items() if k != "leaves"}
    return {"conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan, "scan_step": _exact_scan_step,
            "norm": _exact_norm, "norm_quant": _exact_norm_quant}[case["kind"]](case, s)


def _edges(s):
    """(batch row, first token, end) of each sequence."""
    if s["lengths"] is None:
        return [(i, 0, s["x"].shape[1]) for i in range(s["x"].shape[0])]
    spans, at = [], 0
    for n in s["lengths"]:
        spans.append((0, at, at + n))
        at += n
    return spans


def _exact_conv(case, s):
    width, x = case["width"], s["x"]
    out, finals, inputs, leaves = torch.zeros_like(x), [], [], []
    w, bias = s["weight"].clone().requires_grad_(case["train"]), s["bias"].clone().requires_grad_(case["train"])
    pieces = []
    for i, (row, a, b) in enumerate(_edges(s)):
        xi = x[row, a:b].clone().requires_grad_(case["train"])
        start = (torch.zeros(width - 1, x.shape[2], dtype=x.dtype, device=x.device) if s["initial"] is None
                 else s["initial"][i].clone()).requires_grad_(case["train"])
        held = torch.cat([start, xi])
        pre = bias.expand(b - a, -1)
        for j in range(width):  # j tokens back
            pre = pre + held[width - 1 - j:held.shape[0] - j] * w[:, width - 1 - j]
        pieces.append(pre / (1 + torch.exp(-pre)))
        finals.append(held[held.shape[0] - (width - 1):])
        inputs.append(xi)
        leaves.append(start)
        out[row, a:b] = pieces[-1].detach()
    final = torch.stack(finals)
    if not case["train"]:
        return [out, final]
    loss = (torch.stack(pieces) * s["dout"]).sum() + (final * s["dfinal"]).sum()
    dx, dw, dbias, dstart = (lambda g: (g[:len(inputs)], g[len(inputs)], g[len(inputs) + 1], g[len(inputs) + 2:]))(
        torch.autograd.grad(loss, inputs + [w, bias] + leaves))
    grads = [torch.stack(dx), dw, dbias] + ([torch.stack(dstart)] if s["initial"] is not None else [])
    return [out, final.detach(), *grads]


def _rows(case, s):
    return [(i, i) for i in range(case["batch"])] if s["slots"] is None else list(enumerate(s["slots"].tolist()))


def _exact_conv_step(case, s):
    out, new = torch.zeros_like(s["x"]), s["state_out"].clone()
    for i, slot in _rows(case, s):
        if slot < 0:
            continue
        held = torch.cat([s["state"][slot], s["x"][i][None]])
        pre = s["bias"] + torch.einsum("kc,ck->c", held, s["weight"])
        out[i] = pre / (1 + torch.exp(-pre))
        new[slot] = held[1:]
    return [out, new]


def _exact_scan(case, s):
    x, A, N = s["x"], s["A"], case["state"]
    per = case["channels"] // case["groups"]
    step = torch.logaddexp(s["dt"] + s["dt_bias"], torch.zeros((), dtype=x.dtype, device=x.device))
    u = step * x
    y, finals = torch.zeros_like(x), []
    if not case["train"]:
        for i, (row, a, b) in enumerate(_edges(s)):
            h = torch.zeros(case["channels"], N, dtype=x.dtype, device=x.device) if s["initial"] is None else s["initial"][i]
            for t in range(a, b):
                B, C = (s[k][row, t].repeat_interleave(per, 0) for k in ("B", "C"))
                h = torch.addcmul(u[row, t, :, None] * B, torch.exp(step[row, t, :, None] * A), h)
                y[row, t] = torch.linalg.vecdot(h, C)
            finals.append(h)
        gated = (y + s["D"] * x) * s["z"] / (1 + torch.exp(-s["z"]))
        return [gated, torch.stack(finals)]
    # a training batch: all rows at once, every state kept
    rows, tokens = x.shape[:2]
    if rows * (tokens + 1) * case["channels"] * N * 8 > 24 << 30:
        return None
    states = torch.zeros(tokens + 1, rows, case["channels"], N, dtype=x.dtype, device=x.device)
    if s["initial"] is not None:
        states[0] = s["initial"]
    for t in range(tokens):
        B, C = (s[k][:, t].repeat_interleave(per, 1) for k in ("B", "C"))
        states[t + 1] = torch.exp(step[:, t, :, None] * A) * states[t] + u[:, t, :, None] * B
        y[:, t] = torch.linalg.vecdot(states[t + 1], C)
    sig = 1 / (1 + torch.exp(-s["z"]))
    skip = y + s["D"] * x
    dy = s["dout"] * s["z"] * sig
    dz = s["dout"] * skip * (sig + s["z"] * sig * (1 - sig))
    dx, dstep = dy * s["D"], torch.zeros_like(x)
    dA, dB, dC = torch.zeros_like(A), torch.zeros_like(s["B"]), torch.zeros_like(s["C"])
    g = s["dfinal"]
    for t in reversed(range(tokens)):
        B, C = (s[k][:, t].repeat_interleave(per, 1) for k in ("B", "C"))
        g = g + dy[:, t, :, None] * C
        dC[:, t] = (states[t + 1] * dy[:, t, :, None]).view(rows, -1, per, N).sum(2)
        dB[:, t] = (g * u[:, t, :, None]).view(rows, -1, per, N).sum(2)
        du = torch.linalg.vecdot(g, B)
        g = g * torch.exp(step[:, t, :, None] * A)
        decay = g * states[t]
        dx[:, t] += du * step[:, t]
        dstep[:, t] = du * x[:, t] + torch.linalg.vecdot(decay, A.expand_as(decay))
        dA += (decay * step[:, t, :, None]).sum(0)
    dpre = dstep / (1 + torch.exp(-(s["dt"] + s["dt_bias"])))
    grads = [dx, dpre, dA, dB, dC, (dy * x).sum((0, 1)), dz, dpre.sum((0, 1))] + ([g] if s["initial"] is not None else [])
    return [skip * s["z"] * sig, states[-1].clone(), *grads]


def _exact_scan_step(case, s):
    out, new = torch.zeros_like(s["x"]), s["state_out"].clone()
    per = case["channels"] // case["groups"]
    for i, slot in _rows(case, s):
        if slot < 0:
            continue
        step = torch.logaddexp(s["dt"][i] + s["dt_bias"], torch.zeros_like(s["dt_bias"]))
        B, C = (s[k][i].repeat_interleave(per, 0) for k in ("B", "C"))
        h = torch.exp(step[:, None] * s["A"]) * s["state"][slot] + (step * s["x"][i])[:, None] * B
        out[i] = ((h * C).sum(-1) + s["D"] * s["x"][i]) * s["z"][i] / (1 + torch.exp(-s["z"][i]))
        new[slot] = h
    return [out, new]


def _exact_norm(case, s):
    leaves = [s[k].clone().requires_grad_(True) for k in ("x", "weight", "residual")]
    x, w, residual = leaves
    stream = x + residual
    out = stream / torch.sqrt(stream.square().mean(-1, keepdim=True) + 1e-5) * w
    grads = torch.autograd.grad([out, stream], leaves, [s["dout"], s["dresidual"]])
    return [out.detach(), stream.detach(), *grads]


def _exact_norm_quant(case, s):
    stream = s["x"] + s["residual"]
    rows, width = stream.shape
    group = case["group"] or width
    y = (stream / torch.sqrt(stream.square().mean(-1, keepdim=True) + 1e-5) * s["weight"]).view(rows, -1, group)
    scale = y.abs().amax(-1) / 448
    return [(y / scale[..., None]).view(rows, width), scale, stream]
