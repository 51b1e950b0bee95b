"""The operators around a selective state space layer as a layer uses them: norm with the residual stream, input projection,
short convolution, the projections to B, C and dt, selective scan, output projection; trained, prefilled with packed prompts,
and generating token by token from caches of slots, eagerly and from a captured graph.

Tolerance: both the layer and its plain form in 32 bits are compared with the plain form in 64 bits.  Every operator is within
a few roundings of its value, as the plain form's steps are, so the layer's error (2-norm, relative) may be eight times the
plain form's, and 2^-22 where that has none."""
import pytest
import torch

import ascend_kernel as ak
from operator_checks import conv_plain, norm_plain, scan_plain

pytestmark = pytest.mark.gpu

WIDTH, INNER, STATE, RANK, TAPS = 96, 192, 16, 12, 4
DEPTH = 2


def parameters(seed, dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale):
        return scale * torch.randn(*shape, generator=gen, device="cuda")

    layers = []
    for _ in range(DEPTH):
        steps = 10 ** (-3 + 2 * torch.rand(INNER, generator=gen, device="cuda"))
        layers.append({
            "norm": 1 + normal(WIDTH, scale=0.1), "in": normal(2 * INNER, WIDTH, scale=WIDTH ** -0.5).to(dtype),
            "conv": normal(INNER, TAPS, scale=0.5), "conv_bias": normal(INNER, scale=0.1),
            "select": normal(RANK + 2 * STATE, INNER, scale=INNER ** -0.5).to(dtype),
            "dt": normal(INNER, RANK, scale=RANK ** -0.5).to(dtype), "dt_bias": steps + torch.log(-torch.expm1(-steps)),
            "A": -(torch.arange(1, STATE + 1, device="cuda") * torch.ones(INNER, 1, device="cuda")).contiguous(),
            "D": 1 + normal(INNER, scale=0.1), "out": normal(WIDTH, INNER, scale=INNER ** -0.5).to(dtype)})
    return layers


def split(p, x):
    """x [.., INNER] -> dt, B, C"""
    low, b, c = (x @ p["select"].t()).split([RANK, STATE, STATE], -1)
    return low @ p["dt"].t(), b.unsqueeze(-2), c.unsqueeze(-2)


def run_layers(layers, x, stream, cu=None, states=None, want_states=False):
    """(last sum with the stream, states): prompts of a batch or packed."""
    ends = []
    for i, p in enumerate(layers):
        conv_start, scan_start = (None, None) if states is None else states[i]
        hidden, stream = ak.rms_norm(x, p["norm"], stream)
        inner, gate = (hidden @ p["in"].t()).chunk(2, -1)
        inner, conv_end = ak.short_conv(inner, p["conv"], p["conv_bias"], "silu", conv_start, cu, True)
        dt, b, c = split(p, inner)
        y, scan_end = ak.selective_scan(inner, dt, p["A"], b, c, p["D"], gate, p["dt_bias"], True, scan_start, cu, True)
        x = y @ p["out"].t()
        ends.append((conv_end, scan_end))
    return x + stream, ends


def run_plain(layers, x, stream):
    for p in layers:
        hidden, stream, _ = norm_plain(x, p["norm"], stream, 1e-5)
        inner, gate = (hidden @ p["in"].t()).chunk(2, -1)
        inner = conv_plain(inner, p["conv"], p["conv_bias"], True, inner.new_zeros(inner.shape[0], TAPS - 1, INNER))[0]
        dt, b, c = split(p, inner)
        x = scan_plain(inner, dt, p["A"], b, c, p["D"], gate, p["dt_bias"], True, None)[0] @ p["out"].t()
    return x + stream


def double(layers):
    return [{k: v.detach().double() for k, v in p.items()} for p in layers]


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def within(got, plain, want, what=""):
    mine, theirs = off(got, want), off(plain, want)
    assert mine <= 8 * theirs + 2.0 ** -22, (what, mine, theirs)


def test_training_step():
    layers = parameters(1)
    x, stream = torch.randn(2, 75, WIDTH, device="cuda"), 3 * torch.randn(2, 75, WIDTH, device="cuda")
    upstream = torch.randn(2, 75, WIDTH, device="cuda")

    def leaves_of(ls, *more):
        return [t.requires_grad_(True) for t in (*more, *(v for p in ls for v in p.values()))]

    def step(run, ls, a, b, d):
        leaves = leaves_of(ls, a, b)
        out = run(ls, a, b)
        out = out[0] if isinstance(out, tuple) else out
        return [out.detach(), *torch.autograd.grad(out, leaves, d)]

    want = step(run_plain, double(layers), x.double(), stream.double(), upstream.double())
    plain = step(run_plain, [{k: v.clone() for k, v in p.items()} for p in layers], x.clone(), stream.clone(), upstream)
    got = step(run_layers, layers, x, stream, upstream)
    names = ["out", "dx", "dstream"] + [f"{k} of layer {i}" for i, p in enumerate(layers) for k in p]
    for g, p, w, name in zip(got, plain, want, names):
        within(g, p, w, name)


LENGTHS = [9, 1, 40, 23]


def test_prompts_then_tokens():
    """Packed prompts leave their states in caches; then every sequence takes twelve tokens more, the batch padded to six rows."""
    layers = parameters(2)
    total = [torch.randn(n + 12, WIDTH, device="cuda") for n in LENGTHS]
    with torch.no_grad():
        want = [run_plain(double(layers), t.double()[None], 0.5 * t.double()[None])[0] for t in total]
        plain = [run_plain(layers, t[None], 0.5 * t[None])[0] for t in total]
        packed = torch.cat([t[:n] for t, n in zip(total, LENGTHS)])[None]
        cu = torch.tensor([0] + LENGTHS).cumsum(0).to("cuda", torch.int32)
        out, ends = run_layers(layers, packed, 0.5 * packed, cu)
        slots = torch.tensor([5, 0, 7, 2, -1, -1], dtype=torch.int32, device="cuda")
        conv_cache = torch.zeros(9, DEPTH, TAPS - 1, INNER, device="cuda")  # one for all layers
        scan_cache = torch.zeros(9, DEPTH, INNER, STATE, device="cuda")
        for i, (conv_end, scan_end) in enumerate(ends):
            conv_cache[slots[:4].long(), i] = conv_end
            scan_cache[slots[:4].long(), i] = scan_end

        x = torch.zeros(6, WIDTH, device="cuda")

        def token():
            row, stream = x, 0.5 * x
            for i, p in enumerate(layers):
                hidden, stream = ak.rms_norm(row, p["norm"], stream)
                inner, gate = (hidden @ p["in"].t()).chunk(2, -1)
                inner = ak.short_conv_step(inner, conv_cache[:, i], p["conv"], p["conv_bias"], "silu", slots)
                dt, b, c = split(p, inner)
                y = ak.selective_scan_step(inner, dt, p["A"], b, c, scan_cache[:, i], p["D"], gate, p["dt_bias"], True, slots)
                row = y @ p["out"].t()
            return row + stream

        kept = conv_cache.clone(), scan_cache.clone()
        token()  # once before the capture; its change of the caches is taken back
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            row = token()
        conv_cache.copy_(kept[0])
        scan_cache.copy_(kept[1])
        tokens = []
        for k in range(12):
            x[:4] = torch.stack([t[n + k] for t, n in zip(total, LENGTHS)])
            if k % 2:
                graph.replay()
                tokens.append(row[:4].clone())
            else:
                tokens.append(token()[:4])
        tokens = torch.stack(tokens, 1)
    at = 0
    for s, n in enumerate(LENGTHS):
        within(torch.cat([out[0, at:at + n], tokens[s]]), plain[s], want[s], f"sequence {s}")
        at += n
    untouched = [s for s in range(9) if s not in (5, 0, 7, 2)]
    assert not conv_cache[untouched].any() and not scan_cache[untouched].any()


def test_half_precision_and_an_8_bit_projection():
    """bf16 activations, and the norm's 8-bit output in front of the input projection: the layer runs and stays near the one
    that keeps 32 bits.  The first rounds every activation to 2^-9 (seven of them in a row per layer), the second the
    normed row to 2^-4 of each value: by the root of their number times the rounding's mean square, times four."""
    layers = parameters(3)
    x = torch.randn(1, 50, WIDTH, device="cuda")
    with torch.no_grad():
        want = run_plain(double(layers), x.double(), x.double())
        low = parameters(3, torch.bfloat16)
        out, _ = run_layers(low, x.bfloat16(), x)  # the stream stays in fp32
        assert off(out, want) <= 4 * (7 * DEPTH) ** 0.5 * 2.0 ** -9
        p = layers[0]
        q, scales, stream = ak.rms_norm_quant(x, p["norm"], x, group_size=32)
        hidden = (q.float().unflatten(-1, (-1, 32)) * scales.unsqueeze(-1)).flatten(-2)
        exact = norm_plain(x.double(), p["norm"].double(), x.double(), 1e-5)[0]
        assert off(hidden, exact) <= 2.0 ** -4 and off(hidden @ p["in"].t(), exact @ p["in"].double().t()) <= 2.0 ** -4
