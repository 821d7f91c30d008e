"""The products on operands held in few bits, as cases that can be timed and compared.

A case is a dict of plain values.  `kind` says which operator it goes through:

  gemm_q4   tcec.gemm_q4                  activations times weights kept in 4 bits with a scale for each group along k
  pack_q4   tcec.pack_q4 + unpack_q4      weights brought to 4 bits, and the values that they then stand for
  wgrad_q8  tcec.wgrad_q8                 the gradient of a layer's weights from its input, which was kept in 8 bits
  keep_q8   tcec.pack_q8 + unpack_q8      activations kept in 8 bits, and the values that they then stand for

`m` counts tokens, `n` a layer's outputs, `k` its inputs.  `pad` > 0: the rows of the dense operand lie in a wider matrix.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOKENS = 128  # of one scale in the 8-bit form


def _gemm(m, n, k, dtype, group, out=None, pad=0):
    return {"kind": "gemm_q4", "m": m, "n": n, "k": k, "dtype": dtype, "group": group, "out": out or dtype, "pad": pad}


def _wgrad(m, n, k, dtype, out="f32", pad=0):
    return {"kind": "wgrad_q8", "m": m, "n": n, "k": k, "dtype": dtype, "out": out, "pad": pad}


def _pack(n, k, dtype, group, scale, pad=0):
    return {"kind": "pack_q4", "n": n, "k": k, "dtype": dtype, "group": group, "scale": scale, "pad": pad}


def _keep(m, k, dtype, pad=0):
    return {"kind": "keep_q8", "m": m, "k": k, "dtype": dtype, "pad": pad}


def listed():
    return [
        # One token through a small projection: the latency of a call is what counts.
        dict(_gemm(1, 1024, 1024, "f16", 128), name="q4_one_token_1024"),
        # One token through a square layer of ordinary size: the step that serving repeats.
        dict(_gemm(1, 4096, 4096, "bf16", 128), name="q4_one_token_4096"),
        # One token in FP32, the framework's own type, through the largest square layer: weights beyond the cache.
        dict(_gemm(1, 16384, 16384, "f32", 64), name="q4_one_token_f32_16384"),
        # A few requests decoded together; nothing is a multiple of a tile, small groups.
        dict(_gemm(13, 5000, 7001, "bf16", 32, pad=7), name="q4_ragged_13"),
        # A prompt: as many tokens as make the product a matter of the tensor cores.
        dict(_gemm(1000, 4096, 4096, "bf16", 128), name="q4_prompt_1000"),
        # Weights of a layer brought to 4 bits when a model is loaded.
        dict(_pack(4096, 4096, "f32", 128, "f16"), name="q4_pack_4096"),
        # A small and ragged one, from half-precision weights with small groups.
        dict(_pack(1000, 777, "bf16", 32, "bf16", pad=3), name="q4_pack_ragged"),
        # A layer's input kept for the backward pass.
        dict(_keep(8192, 4096, "bf16"), name="q8_keep_8192"),
        # The same for a short and ragged batch in FP32.
        dict(_keep(1111, 1500, "f32", pad=5), name="q8_keep_ragged"),
        # The gradient of an adapter of rank 16 beside a square layer: each kept value is read for few products.
        dict(_wgrad(8192, 16, 4096, "bf16"), name="q8_wgrad_rank_16"),
        # The gradient of a whole square layer in FP32 from half-precision activations.
        dict(_wgrad(8192, 4096, 4096, "bf16"), name="q8_wgrad_4096"),
        # FP32 throughout, ragged in every direction.
        dict(_wgrad(1111, 777, 1500, "f32", pad=1), name="q8_wgrad_ragged_f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gemm_q4", "gemm_q4", "gemm_q4", "pack_q4", "keep_q8", "wgrad_q8", "wgrad_q8"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    pad = rng.choice([0, 0, 0, 8, rng.randint(1, 40)])
    group = rng.choice([32, 64, 128, 128])

    def width(lo=64, hi=16384):
        v = _log(rng, lo, hi)
        return v if rng.random() < 0.4 else max(8, v // 64 * 64)

    if kind == "gemm_q4":
        while True:  # from one token to long prompts
            m, n, k = _log(rng, 1, 4096), width(), width()
            if m * n * k <= 2**36:
                return _gemm(m, n, k, dtype, group, rng.choice([dtype, dtype, "f32"]), pad)
    if kind == "pack_q4":
        while True:
            n, k = width(), width()
            if n * k <= 2**25:
                return _pack(n, k, dtype, group, rng.choice(["f16", "bf16"]), pad)
    if kind == "keep_q8":
        while True:
            m, k = _log(rng, 1, 16384), width()
            if m * k <= 2**25:
                return _keep(m, k, dtype, pad)
    while True:  # from the rank of an adapter to a whole layer
        m, n, k = _log(rng, 128, 16384), _log(rng, 8, 8192), width()
        if m * n * k <= 2**36 and n * k <= 2**26:
            return _wgrad(m, n, k, dtype, rng.choice(["f32", "f32", dtype]), pad)


def _strided(t, pad):
    """The same values as the left part of a matrix that is `pad` columns wider."""
    if not pad:
        return t
    wide = torch.empty(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _activations(gen, m, k, dtype):
    """Activations: features differ in size, a few of them by a lot, and tokens do so a little."""
    x = torch.randn(m, k, device=DEVICE, generator=gen)
    x *= torch.exp(0.5 * torch.randn(k, device=DEVICE, generator=gen))
    x *= 1 + 15 * (torch.rand(k, device=DEVICE, generator=gen) < 0.005)
    x *= torch.exp(0.2 * torch.randn(m, 1, device=DEVICE, generator=gen))
    return x.to(TYPES[dtype])


def _weights(gen, n, k, dtype):
    w = torch.randn(n, k, device=DEVICE, generator=gen)
    w *= torch.exp(0.3 * torch.randn(n, 1, device=DEVICE, generator=gen)) / math.sqrt(k)
    return w.to(TYPES[dtype])


def _groups(t, size):
    """[rows, k] -> [rows, groups, size], the last group filled with zeros."""
    rows, k = t.shape
    count = -(-k // size)
    if count * size != k:
        t = torch.nn.functional.pad(t, (0, count * size - k))
    return t.reshape(rows, count, size)


def _to_q4(w, group, scale):
    """Codes 0..15 (uint8, n x groups x group), scales in 16 bits and zero points (n x groups)."""
    g = _groups(w.float(), group)
    low, high = g.amin(2).clamp(max=0), g.amax(2).clamp(min=0)
    s = ((high - low).double() / 15).float().to(TYPES[scale])
    d = s.double().clamp(min=1e-30)
    z = torch.round(-low.double() / d).clamp(0, 15)
    q = (torch.round(g.double() / d[:, :, None]) + z[:, :, None]).clamp(0, 15)
    return q.to(torch.uint8), s, z.to(torch.uint8)


def _to_q8(x):
    """Codes -127..127 (int8, m x k) and the FP32 scale of every 128 tokens of a feature (blocks x k)."""
    m, k = x.shape
    blocks = -(-m // TOKENS)
    g = torch.nn.functional.pad(x.float(), (0, 0, 0, blocks * TOKENS - m)).reshape(blocks, TOKENS, k)
    s = (g.abs().amax(1).double() / 127).float().clamp(min=2.0**-120)
    q = torch.round(g.double() / s.double()[:, None, :])
    return q.reshape(blocks * TOKENS, k)[:m].to(torch.int8), s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, state = case["kind"], {"case": dict(case)}
    if kind == "gemm_q4":
        w = _weights(gen, case["n"], case["k"], "f32")
        state["codes"], state["scales"], state["zeros"] = _to_q4(w, case["group"], "f16")
        state["x"] = _strided(_activations(gen, case["m"], case["k"], case["dtype"]), case["pad"])
        if own:
            from wmma_extension_b200 import tcec

            state["packed"] = tcec.pack_q4(w, group=case["group"], scale=torch.float16)
    elif kind == "pack_q4":
        state["w"] = _strided(_weights(gen, case["n"], case["k"], case["dtype"]), case["pad"])
    elif kind == "keep_q8":
        state["x"] = _strided(_activations(gen, case["m"], case["k"], case["dtype"]), case["pad"])
    elif kind == "wgrad_q8":
        x = _activations(gen, case["m"], case["k"], case["dtype"])
        state["codes"], state["scales"] = _to_q8(x)
        # gradients are small, and differ from token to token
        dy = torch.randn(case["m"], case["n"], device=DEVICE, generator=gen)
        dy *= 1e-3 * torch.exp(torch.randn(case["m"], 1, device=DEVICE, generator=gen))
        state["dy"] = _strided(dy.to(TYPES[case["dtype"]]), case["pad"])
        if own:
            from wmma_extension_b200 import tcec

            state["packed"] = tcec.pack_q8(x)
    return state


def _run_own(state):
    from wmma_extension_b200 import tcec

    case = state["case"]
    kind = case["kind"]
    if kind == "gemm_q4":
        return tcec.gemm_q4(state["x"], state["packed"], case["n"], group=case["group"], dtype=TYPES[case["out"]])
    if kind == "pack_q4":
        packed = tcec.pack_q4(state["w"], group=case["group"], scale=TYPES[case["scale"]])
        return tcec.unpack_q4(packed, case["n"], case["k"], group=case["group"])
    if kind == "keep_q8":
        packed = tcec.pack_q8(state["x"])
        return tcec.unpack_q8(packed, case["m"], case["k"])
    return tcec.wgrad_q8(state["dy"], state["packed"], case["k"], dtype=TYPES[case["out"]])


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "gemm_q4":
        q = state["codes"].float() - state["zeros"].float()[:, :, None]
        w = (q * state["scales"].float()[:, :, None]).reshape(case["n"], -1)[:, :case["k"]]
        return (state["x"].float() @ w.T).to(TYPES[case["out"]])
    if kind == "pack_q4":
        q, s, z = _to_q4(state["w"], case["group"], case["scale"])
        w = (q.float() - z.float()[:, :, None]) * s.float()[:, :, None]
        return w.reshape(case["n"], -1)[:, :case["k"]].contiguous()
    if kind == "keep_q8":
        q, s = _to_q8(state["x"])
        return q.float() * s.repeat_interleave(TOKENS, 0)[:case["m"]]
    x = state["codes"].float() * state["scales"].repeat_interleave(TOKENS, 0)[:case["m"]]
    return (state["dy"].float().T @ x).to(TYPES[case["out"]])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "gemm_q4":
        n, k, group = case["n"], case["k"], case["group"]
        out = torch.zeros(case["m"], n, dtype=torch.float64, device=DEVICE)
        for j in range(0, n, 2048):  # some of the weights at a time
            step = state["codes"][j:j + 2048].to(torch.float64)
            step -= state["zeros"][j:j + 2048].to(torch.float64).unsqueeze(2)
            step *= state["scales"][j:j + 2048].to(torch.float64).unsqueeze(2)
            out[:, j:j + 2048] = state["x"].to(torch.float64) @ step.reshape(step.shape[0], -1)[:, :k].t()
        return out
    if kind == "pack_q4":
        w, group = state["w"].to(torch.float64), case["group"]
        n, k = w.shape
        out = torch.empty_like(w)
        for first in range(0, k, group):  # one group of all rows at a time
            part = w[:, first:first + group]
            low = torch.minimum(part.min(dim=1).values, torch.zeros((), dtype=torch.float64, device=DEVICE))
            high = torch.maximum(part.max(dim=1).values, torch.zeros((), dtype=torch.float64, device=DEVICE))
            span = (high - low).to(torch.float32).to(torch.float64)
            scale = (span / 15).to(torch.float32).to(TYPES[case["scale"]]).to(torch.float64)
            some = scale > 0
            step = torch.where(some, scale, torch.ones_like(scale))
            zero = torch.clamp(torch.round(-low / step), 0, 15)
            code = torch.clamp(torch.round(part / step[:, None]) + zero[:, None], 0, 15)
            out[:, first:first + group] = torch.where(some[:, None], (code - zero[:, None]) * scale[:, None], torch.zeros_like(part))
        return out
    if kind == "keep_q8":
        x = state["x"].to(torch.float64)
        out = torch.empty_like(x)
        for first in range(0, x.shape[0], TOKENS):
            part = x[first:first + TOKENS]
            scale = torch.clamp((part.abs().max(dim=0).values / 127).to(torch.float32).to(torch.float64), min=2.0**-120)
            out[first:first + TOKENS] = torch.round(part / scale) * scale
        return out
    out = torch.zeros(case["n"], case["k"], dtype=torch.float64, device=DEVICE)
    for b in range(state["scales"].shape[0]):  # 128 tokens at a time
        rows = slice(b * TOKENS, (b + 1) * TOKENS)
        out += (state["dy"][rows].to(torch.float64).t() @ state["codes"][rows].to(torch.float64)) * state["scales"][b].to(torch.float64)
    return out


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    kind, k = case["kind"], case["k"]
    if kind in ("gemm_q4", "pack_q4"):
        n, groups = case["n"], -(-k // case["group"])
        held = n * k / 2 + n * groups * 2.5  # codes, scales of 16 bits, zero points of 4
    else:
        held = case["m"] * k + -(-case["m"] // TOKENS) * k * 4
    if kind == "gemm_q4":
        m = case["m"]
        return {"bytes": held + m * k * size[case["dtype"]] + m * n * size[case["out"]], "flops": 2.0 * m * n * k}
    if kind == "pack_q4":  # read, held, read again and written out in FP32
        return {"bytes": n * k * size[case["dtype"]] + 2 * held + n * k * 4, "flops": 6.0 * n * k}
    if kind == "keep_q8":
        return {"bytes": case["m"] * k * size[case["dtype"]] + 2 * held + case["m"] * k * 4, "flops": 4.0 * case["m"] * k}
    m, n = case["m"], case["n"]
    return {"bytes": held + m * n * size[case["dtype"]] + n * k * size[case["out"]], "flops": 2.0 * m * n * k}
