"""The 4-bit projection path and the quantized key/value cache, as the framework's operators are
measured on them.

Operators (public entry points in `mcoplib.custom_ops` and `torch.ops._C`):
  quant       mxfp4_quant, its codes read back with mxfp4_dequant: activations or weights in blocks of
              32 values, 4-bit codes (e2m1) and one power-of-two scale (e8m0) a block
  norm_quant  rms_norm_mxfp4_quant: residual add + RMSNorm + the same codes, read back the same way
  mm          mxfp4_scaled_mm: the product of two such operands, with bias and output rounding
  write       kv_cache_write_quant: new keys and values quantized into a paged cache
  read        kv_cache_read_dequant: sequences of that cache gathered and widened
  round_trip  a write, then a read of the tokens it wrote

What is held in 4 bits is compared as the values it stands for: quant, norm_quant and round_trip
include the operator that reads the codes back.  fp8 caches are compared as they are, with their
scales.

Activations are N(0, 1) with 1% of the channels scaled by 20, weights N(0, 0.02), norm weights
N(1, 0.1), keys and values N(0, 1).
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BLOCK = 32  # values that share a scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the activations of a decode step of 16 sequences, before an attention-output projection
        dict(name="quant_t16", op="quant", tokens=16, hidden=5120, dtype="bf16"),
        # prefill of 8192 tokens at a 70B-class width
        dict(name="quant_prefill", op="quant", tokens=8192, hidden=8192, dtype="bf16"),
        # one token of one user: the norm before its QKV projection (the smallest call)
        dict(name="norm_quant_t1", op="norm_quant", tokens=1, hidden=5120, dtype="bf16",
             residual=True),
        # the same before a prefill's projections
        dict(name="norm_quant_prefill", op="norm_quant", tokens=8192, hidden=8192, dtype="bf16",
             residual=True),
        # one token's projection: the weight is read once, nothing else counts
        dict(name="mm_t1", op="mm", m=1, n=8192, k=5120, dtype="bf16", bias=True),
        # a decode step of 64 sequences through a wide up-projection
        dict(name="mm_t64", op="mm", m=64, n=16384, k=5120, dtype="bf16", bias=False),
        # a short prompt and odd sizes: 1237 tokens, 4099 outputs (a vocabulary shard's logits in fp32),
        # 161 blocks a row
        dict(name="mm_ragged", op="mm", m=1237, n=4099, k=5152, dtype="fp32", bias=True),
        # the largest: a prefill of 8192 tokens through a square projection
        dict(name="mm_prefill", op="mm", m=8192, n=8192, k=8192, dtype="bf16", bias=False),
        # a decode step's new token of 64 sequences, 8 key/value heads of 128, fp8 cache
        dict(name="write_t64_fp8", op="write", cache="fp8", tokens=64, heads=8, key=128, value=128,
             page=16, dtype="bf16", fused=True, padded=True),
        # a prefill's 16384 tokens, slices of a fused QKV projection's output
        dict(name="write_prefill_fp8", op="write", cache="fp8", tokens=16384, heads=8, key=128,
             value=128, page=16, dtype="bf16", fused=True, padded=True),
        # the context of 32 running sequences (ragged, 64k tokens) for a chunk's attention, int8 cache
        dict(name="read_context_int8", op="read", cache="int8", tokens=65536, sequences=32, heads=8,
             key=128, value=128, page=16, dtype="bf16", started=True),
        # a 4-bit cache: one prompt of 4096 tokens written and read back, keys wider than values
        dict(name="round_trip_mxfp4", op="round_trip", cache="mxfp4", tokens=4096, sequences=3,
             heads=4, key=192, value=128, page=64, dtype="bf16", fused=False, padded=False,
             started=False),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    """Any operator: 1 to 16384 tokens, widths of 32 to 32768, products of up to 2^39 multiplications,
    caches of 1 to 16 heads of 16 to 256, every type."""
    op = rng.choice(("quant", "norm_quant", "mm", "mm", "write", "read", "round_trip"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op in ("quant", "norm_quant"):
        tokens = _log(rng, 1, 16384)
        hidden = BLOCK * _log(rng, 1, min(1024, max(1, (1 << 26) // (BLOCK * tokens))))
        case = dict(op=op, tokens=tokens, hidden=hidden, dtype=dtype)
        if op == "norm_quant":
            case["residual"] = rng.random() < 0.6
        return case
    if op == "mm":
        while True:
            m, n, k = _log(rng, 1, 16384), _log(rng, 16, 16384), BLOCK * _log(rng, 1, 512)
            if m * n * k <= 1 << 39:
                return dict(op=op, m=m, n=n, k=k, dtype=dtype, bias=rng.random() < 0.5)
    cache = rng.choice(tuple(CACHES)) if op != "write" else "fp8"
    step = BLOCK if cache == "mxfp4" else rng.choice((1, 8, 16))
    width = lambda: step * max(1, _log(rng, 16, 256) // step)  # noqa: E731
    key = width()
    case = dict(op=op, cache=cache, tokens=_log(rng, 1, 32768), heads=rng.randint(1, 16), key=key,
                value=key if rng.random() < 0.6 else width(),
                page=rng.choice((1, 16, 16, 64, 7)), dtype=dtype)
    if op != "read":
        case.update(fused=rng.random() < 0.5, padded=op == "write" and rng.random() < 0.5)
    if op != "write":
        case.update(sequences=rng.randint(1, 64), started=op == "read" and rng.random() < 0.5)
    return case


# ------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)


def _activations(g, tokens, hidden, dtype):
    x = torch.randn(tokens, hidden, generator=g, device="cuda")
    wide = torch.rand(hidden, generator=g, device="cuda") < 0.01
    return (x * torch.where(wide, 20.0, 1.0)).to(dtype)


def _lengths(case, g):
    """Ragged lengths of the case's sequences, some of them empty where there are many tokens a
    sequence to share out, and their first positions."""
    cuts = torch.rand(case["sequences"] - 1, generator=g, device="cuda") * (case["tokens"] + 1)
    edges = torch.cat([cuts.sort().values.to(torch.int32).cpu(),
                       torch.tensor([case["tokens"]], dtype=torch.int32)])
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), edges])
    starts = torch.zeros(case["sequences"], dtype=torch.int32)
    if case["started"]:
        starts = (torch.rand(case["sequences"], generator=g, device="cuda") * 100).to(
            torch.int32).cpu()
    return cu, starts


def _pages(case, g):
    """(block table, cu_seqlens, starts, pages of the cache, slot of every token) of a cache whose
    pages are given out in random order."""
    page = case["page"]
    cu, starts = _lengths(case, g)
    ends = cu[1:] - cu[:-1] + starts
    held = (ends + page - 1) // page
    columns = max(1, int(held.max()))
    pages = int(held.sum()) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(case["sequences"], columns, dtype=torch.int32)
    column = torch.arange(columns).expand_as(table)
    table[column < held[:, None]] = order[:int(held.sum())]
    token = torch.arange(case["tokens"])
    sequence = torch.searchsorted(cu[1:].contiguous(), token.to(torch.int32), right=True)
    at = token - cu[sequence] + starts[sequence]
    slots = table[sequence, at // page].long() * page + at % page
    return table.cuda(), cu.cuda(), starts.cuda(), pages, slots.cuda()


def _empty_cache(case, pages):
    page, heads, kind = case["page"], case["heads"], case["cache"]
    buffers = {}
    for name in ("key", "value"):
        width = case[name]
        codes = width // 2 if kind == "mxfp4" else width
        tail = (width // BLOCK,) if kind == "mxfp4" else ()
        buffers[name + "_cache"] = torch.zeros(pages, page, heads, codes, dtype=CACHES[kind],
                                               device="cuda")
        buffers[name + "_scale"] = torch.zeros(
            pages, page, heads, *tail, device="cuda",
            dtype=torch.uint8 if kind == "mxfp4" else torch.float32)
    return buffers


def _new_tokens(case, g):
    """Keys and values, of their own or as slices of one projection's output beside its queries."""
    heads, key, value, dtype = case["heads"], case["key"], case["value"], DTYPES[case["dtype"]]
    if not case["fused"]:
        return (_randn(g, case["tokens"], heads, key, dtype=dtype),
                _randn(g, case["tokens"], heads, value, dtype=dtype))
    queries = 4 * heads * key
    qkv = _randn(g, case["tokens"], queries + heads * (key + value), dtype=dtype)
    k = qkv[:, queries:queries + heads * key]
    v = qkv[:, queries + heads * key:]
    return k.unflatten(1, (heads, key)), v.unflatten(1, (heads, value))


def prepare(case, seed):
    g = _generator(seed)
    state, op, dtype = dict(case), case["op"], DTYPES[case["dtype"]]
    if op in ("quant", "norm_quant"):
        state["x"] = _activations(g, case["tokens"], case["hidden"], dtype)
        if op == "norm_quant":
            state["weight"] = _randn(g, case["hidden"], scale=0.1, mean=1.0, dtype=dtype)
            if case["residual"]:
                state["running"] = _randn(g, case["tokens"], case["hidden"], dtype=dtype)
    elif op == "mm":
        a = _activations(g, case["m"], case["k"], torch.bfloat16)
        b = _randn(g, case["n"], case["k"], scale=0.02, dtype=torch.bfloat16)
        state["a"], state["a_scale"] = _packed(*_blocks(a))
        state["b"], state["b_scale"] = _packed(*_blocks(b))
        state["bias"] = _randn(g, case["n"], dtype=dtype) if case["bias"] else None
    elif op == "write":
        pages = (case["tokens"] + case["page"] - 1) // case["page"] * 2 + 1
        state.update(_empty_cache(case, pages))
        state["new_key"], state["new_value"] = _new_tokens(case, g)
        slots = torch.randperm(pages * case["page"], generator=g, device="cuda")[:case["tokens"]]
        if case["padded"]:  # a batch padded to a captured size: every 8th token is none
            slots = torch.where(torch.arange(case["tokens"], device="cuda") % 8 == 7, -1, slots)
        state["slots"] = slots
    else:
        table, cu, starts, pages, slots = _pages(case, g)
        state.update(_empty_cache(case, pages), table=table, cu=cu, slots=slots,
                     starts=starts if case["started"] else None)
        if op == "read":
            k = _randn(g, case["tokens"], case["heads"], case["key"], dtype=dtype)
            v = _randn(g, case["tokens"], case["heads"], case["value"], dtype=dtype)
            _write(state, k, v)
        else:
            state["new_key"], state["new_value"] = _new_tokens(case, g)
    return state


# ---------------------------------------------------------------------------------- plain form


def _blocks(x):
    """(codes 0..15, scale bytes) of x in blocks of 32: the largest power of two that leaves a block's
    largest magnitude in [4, 8), to the nearest code, ties to the even one, at most 6."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    most = v.abs().amax(-1)
    byte = torch.where(most == 0, 0, (torch.frexp(most).exponent + 124).clamp_min(0))
    byte = torch.where(torch.isfinite(most), byte, 255)
    q = torch.ldexp(v.abs(), (127 - byte)[..., None])
    code = ((q > 0.25).int() + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5)
            + (q > 5))
    code = code + 8 * torch.signbit(v)
    code = torch.where((byte == 255)[..., None], 0, code)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def _packed(code, byte):
    pairs = code.unflatten(-1, (-1, 2))
    return pairs[..., 0] | (pairs[..., 1] << 4), byte


def _unpacked(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def _block_values(code, byte):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=code.device)
    v = table[code.int()].unflatten(-1, (-1, BLOCK))
    scaled = torch.ldexp(v, (byte.int() - 127)[..., None])
    return torch.where((byte == 255)[..., None], math.nan, scaled).flatten(-2)


def _norm(state):
    """The normalized rows and the new residual: each step rounded once, the sum of squares in 64
    bits."""
    x, dtype = state["x"], state["x"].dtype
    a = x.float()
    if state["residual"]:
        a = a + state["running"].float()
    total = (a.double() * a.double()).sum(-1, keepdim=True).float()
    mean = (total.double() / state["hidden"]).float() + EPS
    rho = (1.0 / mean.double().sqrt().float().double()).float()
    y = ((a * rho).to(dtype).float() * state["weight"].float()).to(dtype)
    return y, (a.to(dtype) if state["residual"] else None)


def _vector_codes(x, kind):
    """(codes as bytes, scales) of each vector along the last dimension."""
    if kind == "mxfp4":
        return _packed(*_blocks(x))
    v = x.float()
    most = v.abs().amax(-1)
    if kind == "int8":
        scale = (most.double() / 127).float()
        inverse = torch.where(most > 0, (127 / most.double()).float(), 0.0)
        code = torch.round(v * inverse[..., None]).clamp(-127, 127).to(torch.int8)
    else:
        scale = (most.double() / 448).float().clamp_min(1.0 / (448.0 * 512.0))
        code = (v / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return code.view(torch.uint8), scale


def _write(state, key, value):
    kept = state["slots"] >= 0
    slots = state["slots"][kept]
    for name, new in (("key", key), ("value", value)):
        code, scale = _vector_codes(new[:kept.numel()][kept], state["cache"])
        state[name + "_cache"].view(torch.uint8).flatten(0, 1)[slots] = code
        state[name + "_scale"].flatten(0, 1)[slots] = scale


def _read(state):
    token = torch.arange(state["tokens"], device="cuda", dtype=torch.int32)
    cu = state["cu"]
    sequence = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    at = token - cu[sequence]
    if state["starts"] is not None:
        at = at + state["starts"][sequence]
    row = state["table"][sequence, at // state["page"]].long() * state["page"] + at % state["page"]
    outs = []
    for name in ("key", "value"):
        code = state[name + "_cache"].flatten(0, 1)[row]
        scale = state[name + "_scale"].flatten(0, 1)[row]
        if state["cache"] == "mxfp4":
            v = _block_values(_unpacked(code), scale)
        else:
            v = code.float() * scale[..., None]
        outs.append(v.to(DTYPES[state["dtype"]]))
    return outs


def _plain(state):
    op = state["op"]
    if op == "quant":
        return _block_values(*_blocks(state["x"])).to(state["x"].dtype)
    if op == "norm_quant":
        y, residual = _norm(state)
        return [_block_values(*_blocks(y)).to(y.dtype)] + ([] if residual is None else [residual])
    if op == "mm":
        a = _block_values(_unpacked(state["a"]), state["a_scale"])
        b = _block_values(_unpacked(state["b"]), state["b_scale"])
        out = a @ b.t()
        if state["bias"] is not None:
            out = out + state["bias"].float()
        return out.to(DTYPES[state["dtype"]])
    if op != "read":
        _write(state, state["new_key"], state["new_value"])
    if op == "write":
        return [state[n] for n in ("key_cache", "value_cache", "key_scale", "value_scale")]
    return _read(state)


# ------------------------------------------------------------------------- the framework's calls


def _cache_of(state):
    return [state[n] for n in ("key_cache", "value_cache", "key_scale", "value_scale")]


def _framework(state):
    from mcoplib import custom_ops

    op = state["op"]
    if op == "quant":
        codes, scales = custom_ops.mxfp4_quant(state["x"])
        return custom_ops.mxfp4_dequant(codes, scales, state["x"].dtype)
    if op == "norm_quant":
        codes, scales, residual = custom_ops.rms_norm_mxfp4_quant(
            state["x"], state["weight"], EPS, state["running"] if state["residual"] else None)
        values = custom_ops.mxfp4_dequant(codes, scales, state["x"].dtype)
        return [values] + ([] if residual is None else [residual])
    if op == "mm":
        return custom_ops.mxfp4_scaled_mm(state["a"], state["a_scale"], state["b"],
                                          state["b_scale"], DTYPES[state["dtype"]], state["bias"])
    if op != "read":
        custom_ops.kv_cache_write_quant(state["new_key"], state["new_value"], *_cache_of(state),
                                        state["slots"])
    if op == "write":
        return _cache_of(state)
    return custom_ops.kv_cache_read_dequant(*_cache_of(state), state["table"], state["cu"],
                                            state["tokens"], DTYPES[state["dtype"]],
                                            state["starts"])


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


# ------------------------------------------------------------------------------ work and exact


def work(case):
    op, b = case["op"], BYTES[case["dtype"]]
    if op in ("quant", "norm_quant"):
        values = case["tokens"] * case["hidden"]
        tensors = 2  # in, and the values of the codes out
        if op == "norm_quant":
            tensors += 2 * case["residual"]  # the residual, in and out
        return {"bytes": values * b * tensors + (case["hidden"] * b if op == "norm_quant" else 0),
                "flops": values * (4 if op == "quant" else 9)}
    if op == "mm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k // 2 + k // BLOCK) + m * n * b + (n * b if case["bias"] else 0),
                "flops": 2 * m * n * k}
    vectors, values = case["tokens"] * case["heads"], case["key"] + case["value"]
    kind = case["cache"]
    held = vectors * (values // 2 + values // BLOCK if kind == "mxfp4" else values + 8)
    plain = vectors * values * b
    if op == "write":
        return {"bytes": (plain + held) * (7 if case["padded"] else 8) // 8 + 8 * case["tokens"],
                "flops": 3 * vectors * values}
    if op == "read":
        return {"bytes": plain + held + 4 * case["tokens"] // case["page"],
                "flops": vectors * values}
    return {"bytes": 2 * plain + held + 8 * case["tokens"], "flops": 4 * vectors * values}


def _exact_blocks(y):
    """The values of y's codes in 64 bits, by the smallest distance over all eight magnitudes; of two
    that are as near the one whose index is even.  A block at a time is scaled by its exponent from
    the logarithm, put right where that is off by one."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=y.device)
    odd = torch.arange(8, device=y.device) % 2 * 1e-9  # a tie goes to the even index
    parts = []
    for part in y.double().split(max(1, (1 << 23) // y.shape[-1])):
        v = part.reshape(*part.shape[:-1], part.shape[-1] // BLOCK, BLOCK)
        most = v.abs().max(-1, keepdim=True).values
        power = torch.floor(torch.log2(most.clamp_min(2.0 ** -126)))
        power = power + (torch.exp2(power + 1) <= most).double() - (torch.exp2(power) > most).double()
        scale = torch.exp2((power - 2).clamp_min(-127.0))
        off = (v.abs().div(scale).unsqueeze(-1) - grid).abs() + odd
        near = grid[off.argmin(-1)] * scale * torch.where(v < 0, -1.0, 1.0)
        parts.append(near.reshape(part.shape))
    return torch.cat(parts)


def _exact_codes(packed, byte):
    """The values of packed codes in 64 bits, from their sign, exponent and fraction bits."""
    both = torch.empty(*packed.shape, 2, dtype=torch.int32, device=packed.device)
    both[..., 0] = packed % 16
    both[..., 1] = packed // 16
    code = both.reshape(*packed.shape[:-1], -1)
    exponent, fraction = (code // 2) % 4, (code % 2).double()
    size = torch.where(exponent > 0, (1 + fraction / 2) * torch.exp2(exponent.double() - 1),
                       fraction / 2)
    power = torch.exp2(byte.double() - 127).repeat_interleave(BLOCK, -1)
    return torch.where(code >= 8, -size, size) * power


def _exact_vectors(x, kind):
    """(the cache's values without their scale, the scales) in 64 bits, the scale, its inverse and the
    scaled value rounded to 32 where the definition rounds them; for 4-bit codes (the values, none)."""
    if kind == "mxfp4":
        return _exact_blocks(x.reshape(-1, x.shape[-1])).reshape(x.shape), None
    v = x.double()
    most = v.abs().max(-1, keepdim=True).values
    if kind == "int8":
        inverse = (127 / most.clamp_min(1e-300)).float().double()
        codes = torch.round((v * inverse).float().double())
        return torch.where(most > 0, codes, 0.0), (most / 127).float().double()
    scale = (most / 448).clamp_min(1 / 229376).float().double()
    q = (v / scale).float().double()
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)  # of e4m3
    return torch.round(q / step) * step, scale


def exact(case, seed):
    state, op, dtype = prepare(case, seed), case["op"], DTYPES[case["dtype"]]
    if op == "quant":
        return _exact_blocks(state["x"])
    if op == "norm_quant":
        # in 64 bits, each result rounded where the operator's definition rounds it: to 32 bits along
        # the row's scalar, to the rows' type at the normalized and at the weighted value
        a = (state["x"].double() + (state["running"].double() if case["residual"] else 0))
        a = a.float().double()
        sums = torch.linalg.vecdot(a, a).float().double()
        mean = (sums / float(case["hidden"])).float()
        root = (mean + torch.tensor(EPS, device="cuda")).double().sqrt().float().double()
        rho = root.reciprocal().float().double().unsqueeze(-1)
        y = (a * rho).float().to(dtype).double() * state["weight"].double()
        y = y.float().to(dtype)
        return [_exact_blocks(y)] + ([a] if case["residual"] else [])
    if op == "mm":
        out = torch.matmul(_exact_codes(state["a"], state["a_scale"]),
                           _exact_codes(state["b"], state["b_scale"]).t().contiguous())
        return out if state["bias"] is None else out + state["bias"].double()
    if op == "write":
        outs = []
        slots = torch.where(state["slots"] < 0, state["key_cache"][:, :, 0, 0].numel(),
                            state["slots"])
        for name in ("key", "value"):
            code, scale = _exact_vectors(state["new_" + name], case["cache"])
            for whole, new in ((state[name + "_cache"], code), (state[name + "_scale"],
                                                               scale.squeeze(-1))):
                flat = torch.zeros(whole.shape[0] * whole.shape[1] + 1, *whole.shape[2:],
                                   dtype=torch.float64, device="cuda")
                flat.index_copy_(0, slots, new)  # padding goes to one row past the cache
                flat[-1] = 0
                outs.append(flat[:-1].reshape(whole.shape))
        return [outs[0], outs[2], outs[1], outs[3]]
    outs = []
    for name in ("key", "value"):
        if op == "round_trip":  # what was written comes back in the same order
            v, scale = _exact_vectors(state["new_" + name], case["cache"])
            outs.append(v if scale is None else v * scale)
            continue
        held, scale = (state[name + s].reshape(-1, *state[name + s].shape[2:])
                       .index_select(0, state["slots"]) if s != "_cache" or case["cache"] != "fp8"
                       else state[name + s].view(torch.uint8).reshape(
                           -1, *state[name + s].shape[2:]).index_select(
                               0, state["slots"]).view(torch.float8_e4m3fn)
                       for s in ("_cache", "_scale"))
        outs.append(_exact_codes(held, scale) if case["cache"] == "mxfp4"
                    else held.double() * scale.double().unsqueeze(-1))
    return outs
