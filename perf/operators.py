"""What is measured of the adapted 4-bit projection's operators.

Three operators, each in its plain form (elementary torch operations in 32 bits, rounded once at
the end) and as the framework's call (`own`):

  matvec / absmax / adapted   products of 1..32 rows with NF4 weights: a span of a layer group
                              (double-quantised scales), a lone projection (fp32 absmax), and a
                              projection with its LoRA adapter in the same call
  dropout                     counter-based dropout and its backward pass, no mask stored
  branch                      the training form of an adapter: dropout, down- and up-projection,
                              added to the base product; forward and backward

The sizes are those of the Qwen2.5-1.5B layer that `qlora` builds (hidden 1536, SwiGLU 8960, key
and value 256), its batch of 4 x 512 tokens, that batch packed (1126 tokens), and odd ones.
"""

import math

import torch

own = False

LEVELS = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453,
          -0.28444138169288635, -0.18477343022823334, -0.09105003625154495, 0.0,
          0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
          0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token through k_proj: the smallest call of a decoding step, all latency
        {"name": "matvec_token_k", "kind": "matvec", "rows": 1, "out": 256, "in": 1536, "bias": True},
        # one token through gate and up as one span: the largest read of a decoding step
        {"name": "matvec_token_gate_up", "kind": "matvec", "rows": 1, "out": 17920, "in": 1536,
         "bias": False},
        # a ragged batch of sequences decoded together, the long reduction of down_proj
        {"name": "matvec_batch_down", "kind": "matvec", "rows": 13, "out": 1536, "in": 8960,
         "bias": False},
        # a projection outside a layer group, odd output size, single-quantised scales
        {"name": "absmax_odd", "kind": "absmax", "rows": 7, "out": 1001, "in": 2112, "block": 128,
         "bias": True},
        # one token through an adapted q_proj: base, bias and adapter in one call
        {"name": "adapted_token_q", "kind": "adapted", "rows": 1, "out": 1536, "in": 1536,
         "rank": 16, "bias": True},
        # the largest batch that the few-row form takes, an adapter of a high rank on down_proj
        {"name": "adapted_batch_down", "kind": "adapted", "rows": 32, "out": 1536, "in": 8960,
         "rank": 64, "bias": False},
        # a short sequence, fp32, columns that are no multiple of anything
        {"name": "dropout_odd_fp32", "kind": "dropout", "rows": 37, "cols": 1537, "dtype": "fp32",
         "p": 0.1},
        # the hidden states of one padded batch at the adapters' own rate
        {"name": "dropout_batch_fp16", "kind": "dropout", "rows": 2048, "cols": 1536,
         "dtype": "fp16", "p": 0.05},
        # the widest activation of a large batch: bandwidth
        {"name": "dropout_wide_bf16", "kind": "dropout", "rows": 16384, "cols": 8960,
         "dtype": "bf16", "p": 0.5},
        # the packed batch through v_proj's adapter
        {"name": "branch_packed_v", "kind": "branch", "rows": 1126, "in": 1536, "out": 256,
         "rank": 16, "p": 0.05},
        # the padded batch through q_proj's adapter: the training step's own case
        {"name": "branch_batch_q", "kind": "branch", "rows": 2048, "in": 1536, "out": 1536,
         "rank": 16, "p": 0.05},
        # a large batch through an adapter of a high rank on up_proj
        {"name": "branch_wide_up", "kind": "branch", "rows": 16384, "in": 1536, "out": 8960,
         "rank": 64, "p": 0.1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["matvec", "absmax", "adapted", "dropout", "branch", "branch"])
    if kind == "dropout":
        rows, cols = _log(rng, 1, 16384), _log(rng, 1, 8960)
        return {"kind": kind, "rows": rows, "cols": cols, "dtype": rng.choice(sorted(DTYPES)),
                "p": round(rng.uniform(0.01, 0.95), 3)}
    if kind == "branch":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "in": 8 * _log(rng, 8, 1120),
                "out": 8 * _log(rng, 8, 192), "rank": rng.choice([1, 4, 8, 12, 16, 16, 32, 64]),
                "p": rng.choice([0.0, 0.05, 0.1, round(rng.uniform(0.01, 0.9), 3)])}
    case = {"kind": kind, "rows": _log(rng, 1, 32), "out": _log(rng, 16, 12000),
            "in": 64 * _log(rng, 1, 140), "bias": rng.random() < 0.5}
    if kind == "absmax":
        case["block"] = rng.choice([64, 64, 128, 256, 1024, 4096])
    if kind == "adapted":
        case["rank"] = rng.choice([1, 4, 8, 16, 16, 32, 64])
    while case["out"] * case["in"] > 17920 * 1536:
        case["out"] = max(16, case["out"] // 3)
    return case


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    kind, rows = case["kind"], case["rows"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    def uniform(*shape, low=0.0, high=1.0):
        return torch.rand(*shape, generator=g, device="cuda") * (high - low) + low

    def codes(n):
        return torch.randint(0, 256, (n,), generator=g, device="cuda", dtype=torch.uint8)

    state = {"kind": kind}
    if kind in ("dropout", "branch"):
        # the seed of one call, drawn as a program draws it from its generator
        state["seed"] = torch.randint(0, 2 ** 62, (1,), generator=g, device="cuda")
        state["p"] = case["p"]
    if kind == "dropout":
        dtype = DTYPES[case["dtype"]]
        state["x"] = normal(rows, case["cols"]).to(dtype).requires_grad_()
        state["g"] = normal(rows, case["cols"], std=0.02).to(dtype)
        return state
    n_in, n_out = case["in"], case["out"]
    if "rank" in case:
        bound = 1.0 / math.sqrt(n_in)  # the adapters' initial A, and a trained B
        state["lora_A"] = uniform(case["rank"], n_in, low=-bound, high=bound)
        state["lora_B"] = normal(n_out, case["rank"], std=0.02)
        state["scaling"] = 2.0
    if kind == "branch":
        state["x"] = normal(rows, n_in).to(torch.float16).requires_grad_()
        state["base"] = normal(rows, n_out).to(torch.float16).requires_grad_()
        state["lora_A"].requires_grad_()
        state["lora_B"].requires_grad_()
        state["g"] = normal(rows, n_out, std=0.02).to(torch.float16)
        return state
    n = n_out * n_in
    state["x"] = normal(rows, n_in).to(torch.float16)
    state["packed"] = codes(n // 2)
    state["bias"] = normal(n_out, std=0.1).to(torch.float16) if case["bias"] else None
    if kind == "absmax":
        state["block"] = case["block"]
        state["absmax"] = uniform(-(-n // case["block"]), low=0.02, high=0.05)
        return state
    # a span that starts behind other projections of its layer, 128 second-level blocks in
    state["row0"], state["qblock"], state["qblock2"] = 128 * 256, 64, 256
    n_rows = n // 64
    n2 = -(-(state["row0"] + n_rows) // 256)
    state["absmax8"] = codes(n_rows)
    code = torch.sort(uniform(256, low=-1.0, high=1.0)).values
    state["code"] = code
    state["absmax2"] = uniform(n2, low=0.2, high=0.4) * 0.035
    state["offset2"] = torch.full((n2,), 0.035, device="cuda")
    state["levels"] = torch.tensor(LEVELS, dtype=torch.float32, device="cuda")
    state["out"] = torch.empty(rows, n_out, dtype=torch.float16, device="cuda")
    return state


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
_LOW = 0xFFFFFFFF


def _round(c0, c1, c2, c3, k0, k1):
    """One round of Philox4x32 on 32-bit values held in int64 (products wrap modulo 2^64)."""
    p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    return (((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW,
            (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW)


def _kept(n, p, seed):
    """The kept elements of n (bool) and the factor they are scaled by."""
    group = torch.arange(-(-n // 8), device=seed.device)
    zero = torch.zeros_like(group)
    v = _round(group & _LOW, group >> 32, zero, zero, seed & _LOW, (seed >> 32) & _LOW)
    v = _round(*_round(*_round(*_round(*_round(*_round(*v))))))
    words = torch.stack(v[:4], 1)
    u = torch.stack((words & 0x7FFF, (words >> 16) & 0x7FFF), 2).reshape(-1)[:n]
    drop = math.floor(p * 32768 + 0.5)
    return u >= drop, 32768.0 / (32768 - drop) if drop < 32768 else 0.0


def _weight(state):
    """The fp32 weight [out, in] of a packed projection."""
    n_in = state["x"].shape[1]
    if state["kind"] == "absmax":
        levels = torch.tensor(LEVELS, dtype=torch.float32, device=state["x"].device)
        scale, block = state["absmax"], state["block"]
    else:
        second = (torch.arange(state["absmax8"].numel(), device=state["x"].device)
                  + state["row0"]) // state["qblock2"]
        scale = (state["code"][state["absmax8"].long()] * state["absmax2"][second]
                 + state["offset2"][second])
        levels, block = state["levels"], state["qblock"]
    byte = state["packed"].long()
    value = levels[torch.stack((byte >> 4, byte & 15), 1).reshape(-1)]
    element = torch.arange(value.numel(), device=value.device)
    return (value * scale[element // block]).view(-1, n_in)


def _plain_matvec(state):
    x = state["x"].float()
    y = x @ _weight(state).t()
    if "lora_A" in state:
        y = y + (x @ state["lora_A"].t()) @ state["lora_B"].t() * state["scaling"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(torch.float16)


def _plain_dropout(state):
    x, g = state["x"], state["g"]
    kept, factor = _kept(x.numel(), state["p"], state["seed"])
    kept = kept.view(x.shape)
    y = torch.where(kept, x.float() * factor, 0.0).to(x.dtype)
    dx = torch.where(kept, g.float() * factor, 0.0).to(x.dtype)
    return {"y": y, "dx": dx}


def _plain_branch(state):
    x, a, b, s = state["x"].float(), state["lora_A"], state["lora_B"], state["scaling"]
    kept, factor = _kept(x.numel(), state["p"], state["seed"])
    kept = kept.view(x.shape)
    g = state["g"].float()
    xd = torch.where(kept, x * factor, 0.0)
    t = xd @ a.t()
    y = (state["base"].float() + t @ b.t() * s).to(torch.float16)
    dt = g @ b * s
    dx = torch.where(kept, (dt @ a) * factor, 0.0).to(torch.float16)
    return {"y": y, "dx": dx, "dA": dt.t() @ xd, "dB": g.t() @ t * s}


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(state):
    kind = state["kind"]
    if not own:
        with torch.no_grad():
            if kind == "dropout":
                return _plain_dropout(state)
            return _plain_branch(state) if kind == "branch" else _plain_matvec(state)
    from talm_b200 import adapter, nf4_dequant, qgroup

    if kind == "dropout":
        x = state["x"]
        y = adapter.dropout(x, state["p"], state["seed"])
        dx, = torch.autograd.grad(y, (x,), state["g"])
        return {"y": y, "dx": dx}
    if kind == "branch":
        leaves = (state["x"], state["lora_A"], state["lora_B"])
        y = adapter.lora_branch(state["x"], state["base"], state["lora_A"], state["lora_B"],
                                state["scaling"], state["p"], state["seed"])
        dx, da, db = torch.autograd.grad(y, leaves, state["g"])
        return {"y": y, "dx": dx, "dA": da, "dB": db}
    if kind == "absmax":
        return nf4_dequant.nf4_matvec(state["x"], state["packed"], state["absmax"],
                                      state["block"], bias=state["bias"])
    extra = (state["lora_A"], state["lora_B"], state["scaling"]) if kind == "adapted" else None
    return qgroup.launch_matvec(state["x"], state["packed"], state["absmax8"], state["code"],
                                state["absmax2"], state["offset2"], state["levels"], state["out"],
                                state["row0"], state["out"].shape[1], state["x"].shape[1],
                                state["qblock"], state["qblock2"], bias=state["bias"],
                                adapter=extra)


# ------------------------------------------------------------------------------------------
# the work of one pass, and its exact result
# ------------------------------------------------------------------------------------------
def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "dropout":
        size = 4 if case["dtype"] == "fp32" else 2
        n = rows * case["cols"]
        return {"bytes": 4 * n * size + 8, "flops": 2 * n}
    n_in, n_out = case["in"], case["out"]
    if kind == "branch":
        r = case["rank"]
        # forward: x, base, A, B read, y written; backward: g, x, A, B read, dx, dA, dB written
        return {"bytes": 2 * rows * (3 * n_in + 3 * n_out) + 12 * r * (n_in + n_out) + 8,
                "flops": 6 * rows * r * (n_in + n_out)}
    n = n_out * n_in
    scales = 4 * -(-n // case["block"]) if kind == "absmax" else n // 64 + 8 * -(-n // (64 * 256))
    r = case.get("rank", 0)
    return {"bytes": n // 2 + scales + 2 * rows * (n_in + n_out) + 4 * r * (n_in + n_out)
            + (2 * n_out if case["bias"] else 0),
            "flops": 2 * rows * n + 2 * rows * r * (n_in + n_out)}


def _exact_kept(n, p, seed):
    """Philox4x32-7 with its products made of 16-bit limbs, so that nothing wraps."""
    group = torch.arange((n + 7) // 8, device=seed.device)
    key = int(seed.item())
    keys = [key % 2 ** 32, (key >> 32) % 2 ** 32]
    c = [group % 2 ** 32, group // 2 ** 32, group * 0, group * 0]

    def product(v, m):
        mid = (v // 65536) * (m % 65536) + ((v % 65536) * (m % 65536)) // 65536
        mid2 = (v % 65536) * (m // 65536) + mid % 65536
        high = (v // 65536) * (m // 65536) + mid // 65536 + mid2 // 65536
        return high, (mid2 % 65536) * 65536 + ((v % 65536) * (m % 65536)) % 65536

    for i in range(7):
        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ ((keys[0] + i * 0x9E3779B9) % 2 ** 32), l1,
             h0 ^ c[3] ^ ((keys[1] + i * 0xBB67AE85) % 2 ** 32), l0]
    u = torch.empty(group.numel(), 8, dtype=torch.int64, device=seed.device)
    for j in range(8):
        u[:, j] = (c[j // 2] // (65536 if j % 2 else 1)) % 32768
    drop = int(p * 32768 + 0.5)
    return u.view(-1)[:n] >= drop, 32768 / (32768 - drop)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64
    with torch.no_grad():
        if kind in ("dropout", "branch"):
            x, g = state["x"].to(f64), state["g"].to(f64)
            kept, factor = _exact_kept(x.numel(), case["p"], state["seed"])
            mask = kept.view(x.shape).to(f64) * factor
            if kind == "dropout":
                return {"y": x * mask, "dx": g * mask}
            a, b = state["lora_A"].to(f64), state["lora_B"].to(f64) * state["scaling"]
            x = x * mask
            t, dt = x @ a.T, g @ b
            return {"y": state["base"].to(f64) + t @ b.T, "dx": (dt @ a) * mask, "dA": dt.T @ x,
                    "dB": state["scaling"] * (g.T @ t)}
        x = state["x"].to(f64)
        n_in, n_out = case["in"], case["out"]
        table = torch.tensor(LEVELS, device="cuda").to(f64)
        codes = torch.empty(n_out, n_in, dtype=torch.int64, device="cuda")
        packed = state["packed"].view(n_out, n_in // 2).to(torch.int64)
        codes[:, 0::2], codes[:, 1::2] = packed // 16, packed % 16
        if kind == "absmax":
            scale = state["absmax"].repeat_interleave(case["block"])[:n_out * n_in]
        else:
            a2 = state["absmax2"].repeat_interleave(256)[state["row0"]:][:n_out * n_in // 64]
            o2 = state["offset2"].repeat_interleave(256)[state["row0"]:][:n_out * n_in // 64]
            # the scale is defined by its two fp32 roundings
            scale = (state["code"][state["absmax8"].to(torch.int64)] * a2 + o2)
            scale = scale.repeat_interleave(64)
        y = x @ (table[codes] * scale.to(f64).view(n_out, n_in)).T
        if "lora_A" in state:
            down = x @ state["lora_A"].to(f64).T
            y = y + state["scaling"] * (down @ state["lora_B"].to(f64).T)
        return y if state["bias"] is None else y + state["bias"].to(f64)
