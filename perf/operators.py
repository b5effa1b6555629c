"""The sequence-mixing, dropout and integer-product operators next to the scan, as cases to measure.

Five kinds of case:

- ``prefill``  attention with a decay for each head over ``[T, B, H, D]`` (chunked form): outputs
               and the final memory
- ``train``    the same with its backward pass: outputs, final memory and every gradient
- ``step``     its recurrent form for one time step over a batch of memories
- ``dropout``  dropout from a counter-based generator, forward and backward
- ``int8``     dense projection in 8-bit integers with a scale for each row and output channel

Where ``own`` is false, ``run`` computes the plain form in elementary torch operations, in 32 bits,
rounded once at the end; where it is true it calls ``myelin_b200``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MAX_ELEMENTS = 256 * 128 * 4096  # the [T, B, N] of the largest scan
MAX_PRODUCT = 51200 * 4096 * 4096  # multiply-adds of the rate network's deep layers
CHUNK = 64  # plain form: time steps per chunk


def listed():
    return [
        # a few new steps on one sequence: the launch and the memory's load are all there is
        {"name": "prefill_small", "kind": "prefill", "T": 8, "B": 1, "H": 4, "Dk": 64, "Dv": 64,
         "dtype": "bf16", "state": True, "ragged": False},
        # one long recording: few (batch, head) rows, so the time axis itself is split
        {"name": "prefill_long", "kind": "prefill", "T": 16384, "B": 1, "H": 16, "Dk": 128,
         "Dv": 128, "dtype": "bf16", "state": True, "ragged": False},
        # a padded batch of prompts, keys narrower than values
        {"name": "prefill_ragged", "kind": "prefill", "T": 1000, "B": 24, "H": 12, "Dk": 64,
         "Dv": 96, "dtype": "f16", "state": False, "ragged": True},
        # the largest training step: the scan's T=256, B=128, N=4096 as 32 heads of 128
        {"name": "train_large", "kind": "train", "T": 256, "B": 128, "H": 32, "Dk": 128, "Dv": 128,
         "dtype": "bf16", "state": False, "ragged": False},
        # a small fp32 model with odd sizes, its memory carried between windows
        {"name": "train_odd_f32", "kind": "train", "T": 333, "B": 5, "H": 7, "Dk": 40, "Dv": 33,
         "dtype": "f32", "state": True, "ragged": True},
        # streaming one sequence, one step at a time
        {"name": "step_one", "kind": "step", "B": 1, "H": 8, "Dk": 64, "Dv": 64, "dtype": "bf16"},
        # serving a full batch of streams
        {"name": "step_batch", "kind": "step", "B": 128, "H": 32, "Dk": 128, "Dv": 128,
         "dtype": "bf16"},
        # dropout on the hidden spikes of the largest scan
        {"name": "dropout_large", "kind": "dropout", "T": 256, "B": 128, "N": 4096, "p": 0.1,
         "dtype": "bf16", "shared": False},
        # one mask for all time steps of a readout's inputs, odd width
        {"name": "dropout_shared", "kind": "dropout", "T": 100, "B": 64, "N": 1001, "p": 0.25,
         "dtype": "f32", "shared": True},
        # one row through a deep layer: the weights' bytes are all there is
        {"name": "int8_row", "kind": "int8", "M": 1, "K": 4096, "N": 4096, "dtype": "bf16",
         "spikes": False},
        # 0/1 spikes through an odd-sized layer
        {"name": "int8_spikes", "kind": "int8", "M": 6400, "K": 784, "N": 1001, "dtype": "bf16",
         "spikes": True},
        # a deep layer of the rate network, all time steps at once
        {"name": "int8_large", "kind": "int8", "M": 51200, "K": 4096, "N": 4096, "dtype": "bf16",
         "spikes": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _head_size(rng):
    """Mostly multiples of 8 between 8 and 128, every fourth any size of that range."""
    return rng.randint(8, 128) if rng.random() < 0.25 else 8 * rng.randint(1, 16)


def draw(rng):
    kind = rng.choice(["prefill", "train", "step", "dropout", "int8"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("prefill", "train"):
        Dk, Dv = _head_size(rng), _head_size(rng)
        H = _log_int(rng, 1, 32)
        most = MAX_ELEMENTS // (8 if kind == "prefill" else 16) // (H * max(Dk, Dv))
        T = _log_int(rng, 1, min(16384, most))
        B = _log_int(rng, 1, max(1, min(128, most // T)))
        return {"kind": kind, "T": T, "B": B, "H": H, "Dk": Dk, "Dv": Dv, "dtype": dtype,
                "state": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    if kind == "step":
        return {"kind": kind, "B": _log_int(rng, 1, 128), "H": _log_int(rng, 1, 32),
                "Dk": _head_size(rng), "Dv": _head_size(rng), "dtype": dtype}
    if kind == "dropout":
        N = _log_int(rng, 16, 4096)
        T = _log_int(rng, 1, 256)
        return {"kind": kind, "T": T, "B": _log_int(rng, 1, 128), "N": N,
                "p": round(rng.uniform(0.05, 0.6), 3), "dtype": dtype,
                "shared": rng.random() < 0.5}
    K, N = _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
    return {"kind": kind, "M": _log_int(rng, 1, 51200), "K": K, "N": N, "dtype": dtype,
            "spikes": rng.random() < 0.3}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        x = torch.empty(shape, dtype=dtype, device="cuda")
        return x.normal_(0.0, std, generator=gen)

    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"kind": kind}
    if kind in ("prefill", "train", "step"):
        B, H, Dk, Dv = (case[n] for n in ("B", "H", "Dk", "Dv"))
        lead = (case["T"], B, H) if kind != "step" else (B, H)
        # time constants of 4 to 512 steps, as decays 1 - 1 / tau
        tau = torch.logspace(2, 9, H, base=2.0, device="cuda", dtype=torch.float64)
        state |= {
            "decay": (1.0 - 1.0 / tau).float(),
            "scale": Dk ** -0.5,
            "q": normal(*lead, Dk, dtype=dtype),
            "k": normal(*lead, Dk, dtype=dtype),
            "v": normal(*lead, Dv, dtype=dtype),
            "lengths": None,
            "memory": None,
        }
        if kind == "step" or case["state"]:
            state["memory"] = normal(B, H, Dk, Dv)
        if kind != "step" and case["ragged"]:
            # real lengths from nothing to the whole window
            T = case["T"]
            state["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device="cuda",
                                             dtype=torch.int32)
            state["lengths"][0] = T
        if kind == "train":
            state["d_out"] = normal(*lead, Dv, dtype=dtype)
            state["d_memory"] = normal(B, H, Dk, Dv) if case["state"] else None
            for name in ("q", "k", "v", "memory"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
    elif kind == "dropout":
        shape = (case["T"], case["B"], case["N"])
        state |= {
            "p": case["p"], "shared": case["shared"],
            "x": normal(*shape, dtype=dtype).requires_grad_(True),
            "d_out": normal(*shape, dtype=dtype),
            "seed": torch.randint(0, 2**62, (2,), generator=gen, device="cuda"),
        }
    else:
        M, K, N = case["M"], case["K"], case["N"]
        if case["spikes"]:
            x = torch.rand((M, K), generator=gen, device="cuda") < 0.2
        else:
            x = normal(M, K, dtype=dtype)
        pitch = (K + 15) // 16 * 16  # weights as a program keeps them: rows of whole 16 bytes
        weight = torch.zeros((N, pitch), dtype=torch.int8, device="cuda")
        weight[:, :K] = torch.randint(-127, 128, (N, K), generator=gen, device="cuda",
                                      dtype=torch.int8)
        state |= {
            "x": x, "weight": weight[:, :K], "dtype": dtype,
            "weight_scale": torch.rand((N,), generator=gen, device="cuda") * 1e-3 + 1e-4,
            "bias": normal(N, dtype=dtype),
        }
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _powers(decay, exponents):
    """decay[h] ** exponents[...], zero where the exponent is negative: [H, ...]."""
    g = decay.view(-1, *([1] * exponents.dim()))
    return torch.where(exponents >= 0, g ** exponents.clamp(min=0), torch.zeros_like(g))


def _heads_first(x, valid=None):
    """[T, B, H, D] as fp32 [B, H, T, D], rows past the lengths replaced by zeros."""
    x = x.detach().float().permute(1, 2, 0, 3)
    return x if valid is None else torch.where(valid[:, None, :, None], x, torch.zeros_like(x))


def _mix(q, k, v, decay, memory, first):
    """sum over j <= i of decay^(i-j) (q_i . k_j) v_j + decay^(i+first) q_i memory, over [B, H, T, D]:
    within chunks from masked scores, between chunks through the memory at each chunk's start."""
    B, H, T, Dk = q.shape
    C, n = CHUNK, (T + CHUNK - 1) // CHUNK
    pad = (0, 0, 0, n * C - T)
    q, k, v = (torch.nn.functional.pad(x, pad).view(B, H, n, C, -1) for x in (q, k, v))
    i = torch.arange(C, device=q.device)
    scores = (q @ k.transpose(-1, -2)) * _powers(decay, i[:, None] - i[None, :])[:, None]
    out = scores @ v
    local = (k * _powers(decay, C - 1 - i)[:, None, :, None]).transpose(-1, -2) @ v
    c = torch.arange(n, device=q.device)
    between = _powers(decay, C * (c[:, None] - 1 - c[None, :]))
    start = (between @ local.flatten(3)).view_as(local)
    out = out + (q * _powers(decay, i + 1)[:, None, :, None]) @ start
    out = out.reshape(B, H, n * C, -1)[:, :, :T]
    if memory is not None:
        t = torch.arange(T, device=q.device)
        whole = q.reshape(B, H, n * C, -1)[:, :, :T] * _powers(decay, t + first)[:, :, None]
        out = out + whole @ memory
    return out


def _gather(k, v, decay, exponents, memory, memory_exponent):
    """sum over j of decay^exponents[b, j] k_j v_j^T + decay^memory_exponent[b] memory."""
    w = _powers(decay, exponents).transpose(0, 1)  # [B, H, T]
    out = (k * w[..., None]).transpose(-1, -2) @ v
    if memory is not None:
        out = out + _powers(decay, memory_exponent).t()[:, :, None, None] * memory
    return out


def _plain_attention(s, backward):
    decay, scale = s["decay"], s["scale"]
    T, B = s["q"].shape[:2]
    dtype = s["q"].dtype
    t = torch.arange(T, device=decay.device)
    if s["lengths"] is None:
        L, valid = torch.full((B,), T, device=decay.device), None
    else:
        L = s["lengths"].long()
        valid = t[None, :] < L[:, None]
    q, k, v = (_heads_first(s[n], valid) for n in ("q", "k", "v"))
    memory = None if s["memory"] is None else s["memory"].detach()

    def rows(x):
        if valid is not None:
            x = torch.where(valid[:, None, :, None], x, torch.zeros_like(x))
        return x.permute(2, 0, 1, 3).contiguous().to(dtype)

    left = L[:, None] - 1 - t[None, :]
    out = {"out": rows(scale * _mix(q, k, v, decay, memory, 1)),
           "memory": _gather(k, v, decay, left, memory, L)}
    if not backward:
        return out
    g, gm = _heads_first(s["d_out"], valid), s["d_memory"]
    out["d_q"] = rows(scale * _mix(g, v, k, decay, None if memory is None
                                   else memory.transpose(-1, -2), 1))
    dk = scale * _mix(v.flip(2), g.flip(2), q.flip(2), decay, None, 0).flip(2)
    dv = scale * _mix(k.flip(2), q.flip(2), g.flip(2), decay, None, 0).flip(2)
    if gm is not None:
        w = _powers(decay, left).transpose(0, 1)[..., None]
        dk = dk + (v * w) @ gm.transpose(-1, -2)
        dv = dv + (k * w) @ gm
        ahead = torch.where(valid, t + 1, -1) if valid is not None else (t + 1).expand(B, T)
        out["d_memory"] = _gather(scale * q, g, decay, ahead, gm, L)
    out["d_k"], out["d_v"] = rows(dk), rows(dv)
    return out


def _plain_step(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    memory = s["decay"][None, :, None, None] * s["memory"] + k[..., :, None] * v[..., None, :]
    out = s["scale"] * (q[..., None, :] @ memory)[..., 0, :]
    return {"out": out.to(s["q"].dtype), "memory": memory}


def _philox(index, seed):
    """Philox 4x32-10 (Salmon et al., 2011): counter (index, offset), key seed; four 32-bit words."""
    mask = 0xFFFFFFFF
    c = [index & mask, (index >> 32) & mask, (seed[1] & mask).expand_as(index),
         ((seed[1] >> 32) & mask).expand_as(index)]
    k0, k1 = seed[0] & mask, (seed[0] >> 32) & mask
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & mask) ^ c[1] ^ k0, b & mask, ((a >> 32) & mask) ^ c[3] ^ k1, a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return c


def _plain_dropout(s):
    x, g = s["x"].detach(), s["d_out"]
    n = x[0].numel() if s["shared"] else x.numel()
    words = torch.stack(_philox(torch.arange((n + 7) // 8, device=x.device), s["seed"]), dim=-1)
    draws = torch.stack([words & 0xFFFF, words >> 16], dim=-1).flatten()[:n]
    threshold = round(s["p"] * 65536)
    keep = (draws >= threshold).view(x.shape[1:] if s["shared"] else x.shape)
    scale = 65536.0 / (65536 - threshold)
    return {"out": torch.where(keep, x.float() * scale, 0.0).to(x.dtype),
            "d_x": torch.where(keep, g.float() * scale, 0.0).to(x.dtype)}


def _plain_int8(s):
    x = s["x"]
    if x.dtype == torch.bool:
        q, row_scale = x.float(), 1.0
    else:
        x = x.float()
        top = x.abs().amax(dim=1, keepdim=True)
        q = torch.round(x * torch.where(top > 0, 127.0 / top, 0.0))
        row_scale = top / 127.0
    y = (q @ s["weight"].float().t()) * (row_scale * s["weight_scale"][None, :])
    return {"out": (y + s["bias"].float()).to(s["dtype"])}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(s):
    import myelin_b200 as mb

    if s["kind"] in ("prefill", "train"):
        first = None if s["memory"] is None else mb.DecayAttentionState(s["memory"])
        last, out = mb.decay_attention_forward(s["q"], s["k"], s["v"], s["decay"], first,
                                               scale=s["scale"], lengths=s["lengths"])
        if s["kind"] == "prefill":
            return {"out": out, "memory": last.memory}
        leaves = [s["q"], s["k"], s["v"]]
        if first is None:
            dq, dk, dv = torch.autograd.grad(out, leaves, s["d_out"])
            return {"out": out, "memory": last.memory, "d_q": dq, "d_k": dk, "d_v": dv}
        dq, dk, dv, dm = torch.autograd.grad((out, last.memory), [*leaves, s["memory"]],
                                             (s["d_out"], s["d_memory"]))
        return {"out": out, "memory": last.memory, "d_q": dq, "d_k": dk, "d_v": dv,
                "d_memory": dm}
    if s["kind"] == "step":
        last, out = mb.decay_attention_step(s["q"], s["k"], s["v"], s["decay"],
                                            mb.DecayAttentionState(s["memory"]),
                                            scale=s["scale"])
        return {"out": out, "memory": last.memory}
    if s["kind"] == "dropout":
        out = mb.spike_dropout(s["x"], s["p"], s["seed"], time_shared=s["shared"])
        (dx,) = torch.autograd.grad(out, [s["x"]], s["d_out"])
        return {"out": out, "d_x": dx}
    weight = mb.QuantizedWeight(s["weight"], s["weight_scale"])
    return {"out": mb.quantized_linear(s["x"], weight, s["bias"], out_dtype=s["dtype"])}


def run(state):
    if own:
        return _own(state)
    if state["kind"] in ("prefill", "train"):
        return _plain_attention(state, state["kind"] == "train")
    return {"step": _plain_step, "dropout": _plain_dropout, "int8": _plain_int8}[state["kind"]](
        state)


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    kind = case["kind"]
    if kind == "dropout":
        n = case["T"] * case["B"] * case["N"]
        return {"bytes": 4 * n * size, "flops": 2 * n}
    if kind == "int8":
        M, K, N = case["M"], case["K"], case["N"]
        read = M * K * (1 if case["spikes"] else size) + N * K + N * (4 + size)
        return {"bytes": read + M * N * size, "flops": 2 * M * N * K}
    B, H, Dk, Dv = (case[n] for n in ("B", "H", "Dk", "Dv"))
    memory = 4 * B * H * Dk * Dv
    rows = B * H * (case["T"] if kind != "step" else 1)
    forward = rows * (2 * Dk + 2 * Dv) * size
    if kind == "step":
        return {"bytes": forward + 2 * memory, "flops": 4 * rows * Dk * Dv}
    states = (2 if case["state"] else 1) * memory
    if kind == "prefill":
        return {"bytes": forward + states, "flops": 4 * rows * Dk * Dv}
    # forward and backward: q, k, v and the outputs' gradient read, outputs and three gradients
    # written; the backward's own products are twice the forward's, and the memory's once more
    backward = rows * (2 * Dk + 2 * Dv) * size
    return {"bytes": forward + backward + (4 if case["state"] else 1) * memory,
            "flops": 14 * rows * Dk * Dv}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_attention(s, backward):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    decay, scale = s["decay"].double()[None, :, None, None], s["scale"]
    T, B, H, Dk = q.shape
    Dv = v.shape[-1]
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    live = torch.tensor([[t < n for n in lengths] for t in range(T)], device=q.device)
    live = live[:, :, None, None]
    # steps past a row's length do nothing: its memory stays and its outputs are zero
    k, q = k.where(live, 0.0), q.where(live, 0.0)
    v = v.where(live, 0.0)
    memory = (torch.zeros((B, H, Dk, Dv), dtype=torch.float64, device=q.device)
              if s["memory"] is None else s["memory"].detach().double().clone())
    out = torch.empty_like(v)
    if backward:
        g = s["d_out"].double().where(live, 0.0)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for t in range(T):
        memory = torch.where(live[t, :, :, :, None], decay * memory, memory)
        memory.addcmul_(k[t][..., :, None], v[t][..., None, :])
        out[t] = scale * torch.einsum("bhd,bhde->bhe", q[t], memory)
        if backward:
            dq[t] = scale * torch.einsum("bhe,bhde->bhd", g[t], memory)
    if not backward:
        return {"out": out, "memory": memory}
    dm = (torch.zeros_like(memory) if s["d_memory"] is None else s["d_memory"].double().clone())
    for t in reversed(range(T)):
        dm.addcmul_(scale * q[t][..., :, None], g[t][..., None, :])
        dk[t] = torch.einsum("bhde,bhe->bhd", dm, v[t])
        dv[t] = torch.einsum("bhde,bhd->bhe", dm, k[t])
        dm = torch.where(live[t, :, :, :, None], decay * dm, dm)
    dk, dv = dk.where(live, 0.0), dv.where(live, 0.0)
    result = {"out": out, "memory": memory, "d_q": dq, "d_k": dk, "d_v": dv}
    if s["d_memory"] is not None:
        result["d_memory"] = dm
    return result


def _times(a, b):
    """High and low 32 bits of a 32-bit tensor times a 32-bit number, by 16-bit halves."""
    a0, a1, b0, b1 = a % 65536, a // 65536, b % 65536, b // 65536
    low, mid1, mid2 = a0 * b0, a1 * b0, a0 * b1
    carry = low // 65536 + mid1 % 65536 + mid2 % 65536
    return a1 * b1 + mid1 // 65536 + mid2 // 65536 + carry // 65536, low % 65536 + carry % 65536 * 65536


def _exact_dropout(s):
    x, g = s["x"].detach().double(), s["d_out"].double()
    n = x[0].numel() if s["shared"] else x.numel()
    seed, offset = (int(w) for w in s["seed"].tolist())
    at = torch.arange(n, device=x.device)
    group, lane = at // 8, at % 8
    w = [group % 2**32, group // 2**32, torch.full_like(group, offset % 2**32),
         torch.full_like(group, offset // 2**32)]
    key = [seed % 2**32, seed // 2**32]
    for _ in range(10):
        h0, l0 = _times(w[0], 0xD2511F53)
        h1, l1 = _times(w[2], 0xCD9E8D57)
        w = [h1 ^ w[1] ^ key[0], l1, h0 ^ w[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    word = torch.where(lane < 2, w[0], torch.where(lane < 4, w[1], torch.where(lane < 6, w[2], w[3])))
    drawn = torch.where(lane % 2 == 0, word % 65536, word // 65536)
    cut = round(s["p"] * 65536)
    factor = torch.where(drawn >= cut, 65536 / (65536 - cut), 0.0).double()
    factor = factor.view(x.shape[1:] if s["shared"] else x.shape)
    return {"out": x * factor, "d_x": g * factor}


def _exact_int8(s):
    x, w = s["x"].double(), s["weight"].double() * s["weight_scale"].double()[:, None]
    if s["x"].dtype != torch.bool:
        step = x.abs().amax(dim=1, keepdim=True) / 127.0
        x = torch.where(step > 0, torch.round(x / step), 0.0) * step
    return {"out": torch.addmm(s["bias"].double(), x, w.t())}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("prefill", "train"):
        return _exact_attention(s, case["kind"] == "train")
    if case["kind"] == "step":
        s["q"], s["k"], s["v"] = (s[n][None] for n in ("q", "k", "v"))
        result = _exact_attention(s, False)
        return {"out": result["out"][0], "memory": result["memory"]}
    return _exact_dropout(s) if case["kind"] == "dropout" else _exact_int8(s)
