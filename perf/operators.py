"""Cases for the sequence operators: the short causal convolution, the selective
state space scan and layer norm, for prompts, training steps and single tokens.

A case names an operator and its sizes.  ``prepare`` makes what a program holds
before the call, ``run`` is one pass, in elementary torch operations or (``own``)
through ``sparsl_b200.Device``; ``exact`` is the definition in 64 bits.

Token arrays are [tokens, channels] with the sequences one after another;
``seq_ptr`` holds where each begins, and rows behind the last one stay as they
were.  States are kept in pools whose row a sequence's ``slots`` entry names.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A batch of prompts of many lengths through one layer's convolution; part of them continue a cached state.
        {"name": "conv prompts packed bf16", "op": "conv", "dtype": "bf16", "tokens": 16384, "seqs": 23, "ragged": True,
         "channels": 4096, "width": 4, "bias": True, "silu": True, "states_kept": True},
        # A training step over unequal documents in full precision, the sequences cut out of longer ones (states in, gradients of states).
        {"name": "conv train odd f32", "op": "conv_train", "dtype": "f32", "tokens": 3001, "seqs": 5, "ragged": True,
         "channels": 1021, "width": 3, "bias": True, "silu": True, "states_kept": True},
        # One new token for each of 64 running sequences.
        {"name": "conv tokens bf16", "op": "conv_token", "dtype": "bf16", "tokens": 64, "channels": 4096, "width": 4,
         "bias": True, "silu": True},
        # One long prompt: nothing but channels and time to work on in parallel.
        {"name": "scan one long bf16", "op": "scan", "dtype": "bf16", "tokens": 32768, "seqs": 1, "ragged": False,
         "channels": 2048, "states": 16, "groups": 1, "gate": True, "states_kept": False},
        # A batch of prompts of many lengths, part of them continued from a cache, states written back in place.
        {"name": "scan prompts packed f16", "op": "scan", "dtype": "f16", "tokens": 12288, "seqs": 19, "ragged": True,
         "channels": 4096, "states": 16, "groups": 1, "gate": True, "states_kept": True},
        # A training step of one layer: the scan and its gradients.
        {"name": "scan train bf16", "op": "scan_train", "dtype": "bf16", "tokens": 16384, "seqs": 8, "ragged": False,
         "channels": 2048, "states": 16, "groups": 1, "gate": True, "states_kept": False},
        # A small odd training step in full precision, two groups of B and C, unequal sequences with states in and their gradients.
        {"name": "scan train odd f32", "op": "scan_train", "dtype": "f32", "tokens": 1531, "seqs": 5, "ragged": True,
         "channels": 402, "states": 11, "groups": 2, "gate": False, "states_kept": True},
        # One new token for a few running sequences: latency.
        {"name": "scan tokens few bf16", "op": "scan_token", "dtype": "bf16", "tokens": 2, "channels": 1024, "states": 16,
         "groups": 1, "gate": True},
        # One new token for each of a large serving batch: the states' traffic.
        {"name": "scan tokens many bf16", "op": "scan_token", "dtype": "bf16", "tokens": 512, "channels": 4096, "states": 16,
         "groups": 1, "gate": True},
        # The norm in front of a layer in training, with its gradients.
        {"name": "norm train bf16", "op": "norm_train", "dtype": "bf16", "tokens": 16384, "channels": 2048},
        # The same in full precision over rows of an odd length.
        {"name": "norm train odd f32", "op": "norm_train", "dtype": "f32", "tokens": 4099, "channels": 5003},
        # The norm of a few new tokens: latency.
        {"name": "norm tokens bf16", "op": "norm", "dtype": "bf16", "tokens": 16, "channels": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "conv_train", "conv_token", "scan", "scan", "scan_train", "scan_train", "scan_token", "norm",
                     "norm_train"])
    c = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op in ("norm", "norm_train"):
        c["channels"] = _log(rng, 33, 12000)
        most = 16384 * 2048 // c["channels"] if op == "norm_train" else 4096
        c["tokens"] = _log(rng, 1, max(2, min(30000, most)))
        return c
    unit = rng.choice([1, 8, 64])
    c["channels"] = max(unit, _log(rng, 48, 6000) // unit * unit)
    if op.endswith("_token"):
        c["tokens"] = _log(rng, 1, max(2, min(600, 512 * 4096 // c["channels"])))
    else:
        most = {"conv": 16384 * 4096, "conv_train": 16384 * 2048, "scan": 16384 * 2048, "scan_train": 8192 * 2048}[op]
        c["tokens"] = _log(rng, 1 if op == "scan" else 16, min(32768, most // c["channels"]))
        c["ragged"] = rng.random() < 0.6
        c["seqs"] = rng.randint(1, max(1, min(40, c["tokens"] // 4)))
        if not c["ragged"]:
            c["tokens"] -= c["tokens"] % c["seqs"]
        c["states_kept"] = rng.random() < 0.5
    if op.startswith("conv"):
        c.update(width=rng.choice([2, 3, 4, 4]), bias=rng.random() < 0.7, silu=rng.random() < 0.7)
    else:
        c.update(states=rng.choice([16, 16, 8, rng.randint(1, 32)]), groups=rng.choice([1, 1, 2, 4]), gate=rng.random() < 0.7)
        c["channels"] = max(1, c["channels"] // c["groups"]) * c["groups"]
        if not op.endswith("_token"):  # more states, fewer tokens: the largest stays the listed one
            keep = max(1, c["tokens"] * 16 // max(16, c["states"]))
            c["seqs"] = min(c["seqs"], keep)
            c["tokens"] = keep if c["ragged"] else keep // c["seqs"] * c["seqs"]
    return c


def _lengths(case, seed):
    """The sequences' lengths: unequal ones leave a few rows behind the last, and hold an empty and a one-token sequence where there are four."""
    n, t = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [t // n] * n
    r = np.random.RandomState(seed % (1 << 31))
    cuts = np.sort(r.randint(0, max(1, t - min(5, t // 2)) + 1, n))
    lens = np.diff(np.concatenate([[0], cuts]))
    if n >= 4 and lens[1] + lens[2] >= 1:
        lens[1], lens[2] = lens[1] + lens[2] - 1, 1
        lens[2], lens[3], lens[0] = 0, 1, lens[0] + lens[3]
    return [int(v) for v in lens]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    f32 = torch.float32
    op, t, ch = case["op"], case["tokens"], case["channels"]

    def normal(*shape, dtype=f32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=gen, device=dev) * (hi - lo) + lo

    s = {"case": dict(case), "stream": torch.cuda.current_stream()}
    if op in ("norm", "norm_train"):
        # Activations with a mean of their own and a few large channels, as residual streams have.
        s["x"] = (normal(t, ch) * (1 + 4 * (uniform(0, 1, ch) > 0.99)) + normal(t, 1) * 0.5).to(dt)
        s["weight"], s["bias"] = (1 + normal(ch, scale=0.1)), normal(ch, scale=0.1)
        s["y"], s["mean"], s["rstd"] = torch.zeros_like(s["x"]), torch.zeros(t, device=dev), torch.zeros(t, device=dev)
        if op == "norm_train":
            s["dy"] = normal(t, ch, dtype=dt)
            s["dx"], s["dweight"], s["dbias"] = torch.zeros_like(s["x"]), torch.zeros(ch, device=dev), torch.zeros(ch, device=dev)
        return s
    # x, and z where there is a gate, are the halves of one projection's output.
    both = normal(t, 2 * ch, dtype=dt)
    s["x"], s["y"] = both[:, :ch], torch.zeros(t, ch, dtype=dt, device=dev)
    token, train = op.endswith("_token"), op.endswith("_train")
    n = t if token else case["seqs"]
    if not token:
        lens = _lengths(case, seed)
        s["lens"] = lens
        s["seq_ptr"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), device=dev) if case["ragged"] else None
        s["seq_ids"] = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(lens, device=dev))
    pool = n + 3
    if token or (case["states_kept"] and not train):
        s["slots"] = torch.randperm(pool, generator=gen, device=dev)[:n].to(torch.int32)
        if not token:
            s["resume"] = (uniform(0, 1, n) < 0.5).to(torch.uint8)
    if op.startswith("conv"):
        w = case["width"]
        s["weight"] = normal(ch, w, scale=1 / math.sqrt(w))
        s["bias"] = normal(ch, scale=0.3) if case["bias"] else None
        shape = (w - 1, ch)
        state_type = dt
    else:
        ns, g = case["states"], case["groups"]
        if case["gate"]:
            s["z"] = both[:, ch:]
        s["dt"] = normal(t, ch, dtype=dt, scale=0.5)
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), ch))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus of it is the step
        s["a"] = -torch.arange(1, ns + 1, device=dev, dtype=f32) * torch.exp(normal(ch, ns, scale=0.2))
        # B and C are slices of the rows of one projection's output, behind the columns that the step sizes come from.
        rows = normal(t, 24 + 2 * g * ns, dtype=dt)
        s["b"], s["c"] = rows[:, 24:24 + g * ns].view(t, g, ns), rows[:, 24 + g * ns:].view(t, g, ns)
        s["d"] = 1 + normal(ch, scale=0.1)
        shape = (ch, ns)
        state_type = f32
    if token:
        s["state"] = normal(pool, *shape, dtype=state_type)
    elif case["states_kept"]:
        s["state"] = normal(n if train else pool, *shape, dtype=state_type)
    if train:
        s["dy"] = normal(t, ch, dtype=dt)
        s["dx"] = torch.zeros(t, ch, dtype=dt, device=dev)
        if case["states_kept"]:
            s["final_state"], s["dfinal_state"] = torch.zeros_like(s["state"]), normal(n, *shape, dtype=state_type, scale=0.3)
            s["dstate"] = torch.zeros_like(s["state"])
        if op == "conv_train":
            s["dweight"] = torch.zeros_like(s["weight"])
            s["dbias"] = torch.zeros(ch, device=dev) if case["bias"] else None
        else:
            s["ddt"] = torch.zeros(t, ch, dtype=dt, device=dev)
            s["db"], s["dc"] = torch.zeros(t, g, ns, dtype=dt, device=dev), torch.zeros(t, g, ns, dtype=dt, device=dev)
            s["da"], s["dd"], s["ddt_bias"] = torch.zeros_like(s["a"]), torch.zeros(ch, device=dev), torch.zeros(ch, device=dev)
            if case["gate"]:
                s["dz"] = torch.zeros(t, ch, dtype=dt, device=dev)
    return s


# ---- the operators in elementary operations, 32 bits, rounded once at the end -----------------


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _initial(s, shape):
    """[seqs, ...]: the state that each sequence starts from, in 32 bits."""
    n = s["case"]["seqs"]
    if "state" not in s:
        return torch.zeros(n, *shape, device="cuda")
    rows = s["state"][s["slots"].long()] if "slots" in s else s["state"]
    rows = rows.float()
    if "resume" in s:
        rows = torch.where(s["resume"].view(n, *([1] * len(shape))) != 0, rows, torch.zeros_like(rows))
    return rows


def _put_final(s, rows):
    to = s.get("final_state", s["state"])
    if "slots" in s:
        to[s["slots"].long()] = rows.to(to.dtype)
    else:
        to.copy_(rows)
    return to


def _spans(s):
    """(first token, token behind the last) of each sequence, on the device."""
    n, t = s["case"]["seqs"], s["case"]["tokens"]
    ptr = s["seq_ptr"].long() if s["seq_ptr"] is not None else torch.arange(n + 1, device="cuda") * (t // n)
    return ptr[:-1], ptr[1:]


def _conv_taps(s):
    """The inputs under the convolution's taps, [used, width, channels], the starts [seqs, width - 1, channels], and each token's place in (start, inputs)."""
    w, ch = s["case"]["width"], s["case"]["channels"]
    first, last = _spans(s)
    n, used = s["case"]["seqs"], s["seq_ids"].numel()
    start = _initial(s, (w - 1, ch))
    x = s["x"][:used].float()
    every = torch.cat([start.reshape(n * (w - 1), ch), x])  # the starts' rows, then the tokens'
    pos = torch.arange(used, device="cuda") - first[s["seq_ids"]]
    at = pos[:, None] - (w - 1) + torch.arange(w, device="cuda")  # place in the sequence of each tap
    at = torch.where(at >= 0, n * (w - 1) + first[s["seq_ids"]][:, None] + at, s["seq_ids"][:, None] * (w - 1) + (w - 1) + at)
    return every, at, first, last


def _conv_final(s, every, first, last):
    """The last width - 1 inputs of each sequence, with those of its start in front."""
    w, n = s["case"]["width"], s["case"]["seqs"]
    at = (last - first)[:, None] - (w - 1) + torch.arange(w - 1, device="cuda")
    seq = torch.arange(n, device="cuda")[:, None]
    return torch.where(at >= 0, n * (w - 1) + first[:, None] + at, seq * (w - 1) + (w - 1) + at)


def _plain_conv(s):
    case = s["case"]
    every, at, first, last = _conv_taps(s)
    u = (every[at] * s["weight"].t()[None]).sum(1)
    if s["bias"] is not None:
        u = u + s["bias"]
    s["y"][:at.shape[0]] = (u * _sigmoid(u) if case["silu"] else u).to(s["y"].dtype)
    out = {"y": s["y"]}
    if "state" in s:
        out["state"] = _put_final(s, every[_conv_final(s, every, first, last)])
    if case["op"] == "conv":
        return out
    du = s["dy"][:at.shape[0]].float()
    if case["silu"]:
        g = _sigmoid(u)
        du = du * g * (1 + u * (1 - g))
    dtap = du[:, None, :] * s["weight"].t()[None]
    every_grad = torch.zeros_like(every)
    every_grad.index_add_(0, at.reshape(-1), dtap.reshape(-1, case["channels"]))
    if "dfinal_state" in s:
        every_grad.index_add_(0, _conv_final(s, every, first, last).reshape(-1), s["dfinal_state"].float().reshape(-1, case["channels"]))
    cut = case["seqs"] * (case["width"] - 1)
    s["dx"][:at.shape[0]] = every_grad[cut:].to(s["dx"].dtype)
    s["dweight"].copy_((every[at] * du[:, None, :]).sum(0).t())
    out.update(dx=s["dx"], dweight=s["dweight"])
    if s["bias"] is not None:
        s["dbias"].copy_(du.sum(0))
        out["dbias"] = s["dbias"]
    if "dstate" in s:
        s["dstate"].copy_(every_grad[:cut].view_as(s["dstate"]))
        out["dstate"] = s["dstate"]
    return out


def _plain_conv_token(s):
    rows = s["slots"].long()
    taps = torch.cat([s["state"][rows], s["x"][:, None, :]], 1)
    u = (taps.float() * s["weight"].t()[None]).sum(1)
    if s["bias"] is not None:
        u = u + s["bias"]
    s["y"].copy_(u * _sigmoid(u) if s["case"]["silu"] else u)
    s["state"][rows] = taps[:, 1:]
    return {"y": s["y"], "state": s["state"]}


def _running(decay, add, longest):
    """h[t] = decay[t] h[t-1] + add[t] along the first axis, by doubling; a decay of zero starts anew."""
    step = 1
    while step < longest:
        more, d = add.clone(), decay.clone()
        more[step:] += decay[step:] * add[:-step]
        d[step:] *= decay[:-step]
        decay, add, step = d, more, 2 * step
    return add


def _softplus(u):
    return torch.clamp(u, min=0) + torch.log1p(torch.exp(-u.abs()))


def _plain_scan(s):
    case = s["case"]
    ch, ns, g = case["channels"], case["states"], case["groups"]
    used, ids = s["seq_ids"].numel(), s["seq_ids"]
    first, last = _spans(s)
    full = last > first
    x = s["x"][:used].float()
    u = s["dt"][:used].float() + s["dt_bias"]
    step = _softplus(u)
    b = s["b"][:used].float().repeat_interleave(ch // g, 1)  # [used, channels, states]
    c = s["c"][:used].float().repeat_interleave(ch // g, 1)
    start = _initial(s, (ch, ns))
    decay = torch.exp(step[:, :, None] * s["a"])
    begins = torch.zeros(used, dtype=torch.bool, device="cuda")
    begins[first[full]] = True
    add = (step * x)[:, :, None] * b
    add[first[full]] += decay[first[full]] * start[full]
    cut = torch.where(begins[:, None, None], torch.zeros_like(decay), decay)
    h = _running(cut, add, max(s["lens"]))
    y = (h * c).sum(2) + s["d"] * x
    if case["gate"]:
        z = s["z"][:used].float()
        sig = _sigmoid(z)
        s["y"][:used] = (y * z * sig).to(s["y"].dtype)
    else:
        s["y"][:used] = y.to(s["y"].dtype)
    out = {"y": s["y"]}
    if "state" in s:
        final = start.clone()
        final[full] = h[last[full] - 1]
        out["state"] = _put_final(s, final)
    if case["op"] == "scan":
        return out
    dy = s["dy"][:used].float()
    if case["gate"]:
        s["dz"][:used] = (dy * y * sig * (1 + z * (1 - sig))).to(s["dz"].dtype)
        out["dz"] = s["dz"]
        dy = dy * z * sig
    into = dy[:, :, None] * c
    if "dfinal_state" in s:
        into[last[full] - 1] += s["dfinal_state"][full]
    after = torch.cat([decay[1:], torch.zeros_like(decay[:1])])  # the decay between a token and the next of its sequence
    after[:-1][begins[1:]] = 0
    grad = _running(after.flip(0), into.flip(0), max(s["lens"])).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first[full]] = start[full]
    through = grad * decay * before
    gb = (grad * b).sum(2)
    s["dx"][:used] = (s["d"] * dy + step * gb).to(s["dx"].dtype)
    du = ((through * s["a"]).sum(2) + x * gb) * _sigmoid(u)
    s["ddt"][:used] = du.to(s["ddt"].dtype)
    s["da"].copy_((through * step[:, :, None]).sum(0))
    s["dd"].copy_((dy * x).sum(0))
    s["ddt_bias"].copy_(du.sum(0))
    s["db"][:used] = (grad * (step * x)[:, :, None]).view(used, g, ch // g, ns).sum(2).to(s["db"].dtype)
    s["dc"][:used] = (h * dy[:, :, None]).view(used, g, ch // g, ns).sum(2).to(s["dc"].dtype)
    out.update({k: s[k] for k in ("dx", "ddt", "da", "db", "dc", "dd", "ddt_bias")})
    if "dstate" in s:
        s["dstate"].copy_(s["dfinal_state"])
        s["dstate"][full] = grad[first[full]] * decay[first[full]]
        out["dstate"] = s["dstate"]
    return out


def _plain_scan_token(s):
    case = s["case"]
    per = case["channels"] // case["groups"]
    rows = s["slots"].long()
    x = s["x"].float()
    step = _softplus(s["dt"].float() + s["dt_bias"])
    b, c = s["b"].float().repeat_interleave(per, 1), s["c"].float().repeat_interleave(per, 1)
    h = torch.exp(step[:, :, None] * s["a"]) * s["state"][rows] + (step * x)[:, :, None] * b
    y = (h * c).sum(2) + s["d"] * x
    if case["gate"]:
        z = s["z"].float()
        y = y * z * _sigmoid(z)
    s["y"].copy_(y)
    s["state"][rows] = h
    return {"y": s["y"], "state": s["state"]}


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + 1e-5)
    hat = (x - mean) * rstd
    s["y"].copy_(hat * s["weight"] + s["bias"])
    s["mean"].copy_(mean[:, 0])
    s["rstd"].copy_(rstd[:, 0])
    out = {k: s[k] for k in ("y", "mean", "rstd")}
    if s["case"]["op"] == "norm":
        return out
    dy = s["dy"].float()
    wd = dy * s["weight"]
    s["dx"].copy_(rstd * (wd - wd.mean(1, keepdim=True) - hat * (wd * hat).mean(1, keepdim=True)))
    s["dweight"].copy_((dy * hat).sum(0))
    s["dbias"].copy_(dy.sum(0))
    out.update({k: s[k] for k in ("dx", "dweight", "dbias")})
    return out


# ---- the framework's calls ----------------------------------------------------------------------

_opened = []


def _device():
    if not _opened:
        import sparsl_b200

        _opened.append(sparsl_b200.Device.try_new(sparsl_b200.Backend.Cuda))
    return _opened[0]


def _room(s, key, size):
    """A workspace that the program keeps beside the buffers, made on the first pass."""
    if key not in s:
        s[key] = torch.empty(max(size(), 1), dtype=torch.uint8, device="cuda")
    return s[key]


def _seqs(s):
    if s["seq_ptr"] is not None:
        return {"seq_ptr": s["seq_ptr"]}
    return {"n_seq": s["case"]["seqs"]}


def _kept(s):
    """The state's arguments of a prompt: its pool is updated in place."""
    if "state" not in s:
        return {}
    return {"state": s["state"], "final_state": s["state"], "slots": s["slots"], "resume": s["resume"]}


def _own(s):
    dev, case, st = _device(), s["case"], s["stream"]
    op, t, ch = case["op"], case["tokens"], case["channels"]
    out = {"y": s["y"]}
    if op == "conv":
        dev.causal_conv_device(s["x"], s["weight"], s["y"], bias=s["bias"], silu=case["silu"], **_seqs(s), **_kept(s), stream=st)
    elif op == "conv_train":
        state, final = s.get("state"), s.get("final_state")
        dev.causal_conv_device(s["x"], s["weight"], s["y"], bias=s["bias"], silu=case["silu"], **_seqs(s), state=state,
                               final_state=final, stream=st)
        room = _room(s, "room", lambda: dev.causal_conv_backward_workspace(t, ch, case["width"]))
        dev.causal_conv_backward_device(s["dy"], s["x"], s["weight"], s["dx"], s["dweight"], room, bias=s["bias"],
                                        dbias=s["dbias"], silu=case["silu"], **_seqs(s), state=state, dstate=s.get("dstate"),
                                        dfinal_state=s.get("dfinal_state"), stream=st)
        out.update(dx=s["dx"], dweight=s["dweight"])
        if s["bias"] is not None:
            out["dbias"] = s["dbias"]
    elif op == "conv_token":
        dev.causal_conv_step_device(s["x"], s["weight"], s["y"], s["state"], bias=s["bias"], silu=case["silu"], slots=s["slots"],
                                    stream=st)
    elif op == "scan":
        room = _room(s, "room", lambda: dev.selective_scan_workspace(t, ch, case["states"], case["seqs"], case["groups"]))
        dev.selective_scan_device(s["x"], s["dt"], s["a"], s["b"], s["c"], s["y"], room, d=s["d"], z=s.get("z"),
                                  dt_bias=s["dt_bias"], softplus=True, **_seqs(s), **_kept(s), stream=st)
    elif op == "scan_train":
        state, final = s.get("state"), s.get("final_state")
        room = _room(s, "room", lambda: max(
            dev.selective_scan_workspace(t, ch, case["states"], case["seqs"], case["groups"]),
            dev.selective_scan_backward_workspace(t, ch, case["states"], case["seqs"], case["groups"])))
        marks = _room(s, "marks", lambda: dev.selective_scan_checkpoints(t, ch, case["states"]))
        dev.selective_scan_device(s["x"], s["dt"], s["a"], s["b"], s["c"], s["y"], room, d=s["d"], z=s.get("z"),
                                  dt_bias=s["dt_bias"], softplus=True, **_seqs(s), state=state, final_state=final,
                                  checkpoints=marks, stream=st)
        dev.selective_scan_backward_device(s["dy"], s["x"], s["dt"], s["a"], s["b"], s["c"], marks, s["dx"], s["ddt"], s["da"],
                                           s["db"], s["dc"], room, d=s["d"], dd=s["dd"], z=s.get("z"), dz=s.get("dz"),
                                           dt_bias=s["dt_bias"], ddt_bias=s["ddt_bias"], softplus=True, **_seqs(s), state=state,
                                           dstate=s.get("dstate"), dfinal_state=s.get("dfinal_state"), stream=st)
        out.update({k: s[k] for k in ("dx", "ddt", "da", "db", "dc", "dd", "ddt_bias")})
        if "dz" in s:
            out["dz"] = s["dz"]
    elif op == "scan_token":
        dev.selective_scan_step_device(s["x"], s["dt"], s["a"], s["b"], s["c"], s["y"], s["state"], d=s["d"], z=s.get("z"),
                                       dt_bias=s["dt_bias"], softplus=True, slots=s["slots"], stream=st)
    else:
        dev.layer_norm_device(s["x"], s["y"], weight=s["weight"], bias=s["bias"], eps=1e-5, mean=s["mean"], rstd=s["rstd"], stream=st)
        out.update(mean=s["mean"], rstd=s["rstd"])
        if op == "norm_train":
            room = _room(s, "room", lambda: dev.layer_norm_backward_workspace(t, ch))
            dev.layer_norm_backward_device(s["dy"], s["x"], s["mean"], s["rstd"], s["dx"], room, weight=s["weight"],
                                           dweight=s["dweight"], dbias=s["dbias"], stream=st)
            out.update({k: s[k] for k in ("dx", "dweight", "dbias")})
        return out
    if "state" in s:
        out["state"] = s.get("final_state", s["state"])
        if "dstate" in s:
            out["dstate"] = s["dstate"]
    return out


_PLAIN = {"conv": _plain_conv, "conv_train": _plain_conv, "conv_token": _plain_conv_token, "scan": _plain_scan,
          "scan_train": _plain_scan, "scan_token": _plain_scan_token, "norm": _plain_norm, "norm_train": _plain_norm}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    op, t, ch = case["op"], case["tokens"], case["channels"]
    e = 4 if case["dtype"] == "f32" else 2
    cell = t * ch
    if op in ("norm", "norm_train"):
        if op == "norm":
            return {"bytes": 2 * cell * e + 8 * t + 8 * ch, "flops": 8 * cell}
        return {"bytes": 4 * cell * e + 8 * t + 16 * ch, "flops": 24 * cell}
    n = t if op.endswith("_token") else case["seqs"]
    kept = op.endswith("_token") or case["states_kept"]
    if op.startswith("conv"):
        w = case["width"]
        state = n * (w - 1) * ch * e if kept else 0
        f = (2 * w + 8) * cell
        if op == "conv_train":
            return {"bytes": 4 * cell * e + 4 * state + 8 * (w + 1) * ch, "flops": 3 * f}
        return {"bytes": 2 * cell * e + 2 * state + 4 * (w + 1) * ch, "flops": f}
    ns, g = case["states"], case["groups"]
    state = n * ch * ns * 4 if kept else 0
    rows = 2 * t * g * ns * e
    gate = 1 if case["gate"] else 0
    f = cell * (7 * ns + 20)
    if op == "scan_train":
        return {"bytes": (6 + 2 * gate) * cell * e + 2 * rows + 4 * state + 8 * ch * (ns + 2), "flops": cell * (30 * ns + 60)}
    return {"bytes": (3 + gate) * cell * e + rows + 2 * state + 4 * ch * (ns + 2), "flops": f}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def _exact_start(s, n):
    if "state" not in s:
        return None
    rows = s["state"].double()
    if "slots" in s:
        rows = rows[s["slots"].long()]
    if "resume" in s:
        rows = rows * s["resume"].double().view(n, 1, 1)
    return rows


def _exact_state(s, rows):
    to = s.get("final_state", s["state"]).double().clone()
    if "slots" in s:
        to[s["slots"].long()] = rows
        return to
    return rows


def _exact_conv(s):
    """Sequence by sequence and tap by tap over the padded sequence, and its transpose."""
    case = s["case"]
    w, ch, train = case["width"], case["channels"], case["op"] == "conv_train"
    weight = s["weight"].double()
    bias = s["bias"].double() if s["bias"] is not None else torch.zeros(ch, dtype=torch.float64, device="cuda")
    x = s["x"].double()
    start = _exact_start(s, case["seqs"])
    y = torch.zeros(case["tokens"], ch, dtype=torch.float64, device="cuda")
    dx, dweight, dbias = torch.zeros_like(y), torch.zeros_like(weight), torch.zeros_like(bias)
    finals, dstarts, at = [], [], 0
    for i, length in enumerate(s["lens"]):
        begin = start[i] if start is not None else torch.zeros(w - 1, ch, dtype=torch.float64, device="cuda")
        line = torch.cat([begin, x[at:at + length]])
        u = bias.expand(length, ch).clone()
        for k in range(w):
            u += weight[:, k] * line[k:k + length]
        y[at:at + length] = u / (1 + torch.exp(-u)) if case["silu"] else u
        finals.append(line[length:])
        if train:
            du = s["dy"][at:at + length].double()
            if case["silu"]:
                g = torch.sigmoid(u)
                du = du * (g + u * g * (1 - g))
            dline = torch.zeros_like(line)
            if "dfinal_state" in s:
                dline[length:] += s["dfinal_state"][i].double()
            for k in range(w):
                dline[k:k + length] += weight[:, k] * du
                dweight[:, k] += (du * line[k:k + length]).sum(0)
            dbias += du.sum(0)
            dx[at:at + length] = dline[w - 1:]
            dstarts.append(dline[:w - 1])
        at += length
    out = {"y": y}
    if start is not None:
        out["state"] = _exact_state(s, torch.stack(finals))
    if train:
        out.update(dx=dx, dweight=dweight)
        if s["bias"] is not None:
            out["dbias"] = dbias
        if "dstate" in s:
            out["dstate"] = torch.stack(dstarts)
    return out


def _exact_scan(s):
    """Token by token, all sequences side by side (the shorter ones wait at their ends); the gradients token by token backwards."""
    case = s["case"]
    ch, ns, g, n = case["channels"], case["states"], case["groups"], case["seqs"]
    f64 = torch.float64
    lens = torch.tensor(s["lens"], device="cuda")
    longest = max(s["lens"])
    first = torch.cumsum(lens, 0) - lens
    grid = first[None] + torch.arange(longest, device="cuda")[:, None]  # [longest, seqs]
    live = torch.arange(longest, device="cuda")[:, None] < lens[None]
    grid = torch.where(live, grid, torch.zeros_like(grid))
    a = s["a"].double()
    u = s["dt"].double() + s["dt_bias"].double()
    step = torch.where(u > 30, u, torch.log1p(torch.exp(torch.clamp(u, max=30))))
    x, b, c = s["x"].double(), s["b"].double(), s["c"].double()
    wide = lambda rows: rows.repeat_interleave(ch // g, 1)  # noqa: E731
    h = _exact_start(s, n)
    h = torch.zeros(n, ch, ns, dtype=f64, device="cuda") if h is None else h.clone()
    start = h.clone()
    pre = torch.zeros(case["tokens"], ch, dtype=f64, device="cuda")
    train = case["op"] == "scan_train"
    kept = []
    for k in range(longest):
        at, m = grid[k], live[k][:, None, None]
        new = torch.exp(step[at][:, :, None] * a) * h + (step[at] * x[at])[:, :, None] * wide(b[at])
        h = torch.where(m, new, h)
        if train:
            kept.append(h)
        o = (new * wide(c[at])).sum(2)
        if n == 1:
            pre[k] = o[0]
        else:
            pre.index_add_(0, at, o * live[k][:, None])
    used = int(lens.sum())
    pre[:used] += s["d"].double() * x[:used]
    out = {}
    z = s["z"].double() if case["gate"] else None
    out["y"] = pre * z * torch.sigmoid(z) if case["gate"] else pre
    if "state" in s:
        out["state"] = _exact_state(s, h)
    if not train:
        return out
    dy = s["dy"].double()
    dy[used:] = 0
    if case["gate"]:
        sig = torch.sigmoid(z)
        out["dz"] = dy * pre * (sig + z * sig * (1 - sig))
        dy = dy * z * sig
    dx, du = s["d"].double() * dy, torch.zeros_like(dy)
    db, dc = torch.zeros_like(b), torch.zeros_like(c)
    da = torch.zeros_like(a)
    grad = s["dfinal_state"].double() if "dfinal_state" in s else torch.zeros_like(h)
    for k in range(longest - 1, -1, -1):
        at, m = grid[k], live[k][:, None, None]
        before = kept[k - 1] if k else start
        now = grad + dy[at][:, :, None] * wide(c[at])
        decay = torch.exp(step[at][:, :, None] * a)
        now = torch.where(m, now, torch.zeros_like(now))
        gb = (now * wide(b[at])).sum(2)
        t = now * decay * before
        da += (t * step[at][:, :, None]).sum(0)
        dx.index_add_(0, at, step[at] * gb)
        du.index_add_(0, at, (t * a).sum(2) + x[at] * gb)
        db.index_add_(0, at, (now * (step[at] * x[at])[:, :, None]).view(n, g, ch // g, ns).sum(2))
        dc.index_add_(0, at, (torch.where(m, kept[k], torch.zeros_like(h)) * dy[at][:, :, None]).view(n, g, ch // g, ns).sum(2))
        grad = torch.where(m, now * decay, grad)
    du = du * torch.sigmoid(u)
    out.update(dx=dx, ddt=du, da=da, db=db, dc=dc, dd=(dy * x)[:used].sum(0), ddt_bias=du.sum(0))
    if "dstate" in s:
        out["dstate"] = grad
    return out


def _exact_token(s):
    case = s["case"]
    rows = s["slots"].long()
    state = s["state"].double().clone()
    x = s["x"].double()
    if case["op"] == "conv_token":
        u = x * s["weight"][:, -1].double()
        for k in range(case["width"] - 1):
            u = u + state[rows, k] * s["weight"][:, k].double()
        if s["bias"] is not None:
            u = u + s["bias"].double()
        y = u * torch.sigmoid(u) if case["silu"] else u
        state[rows] = torch.cat([state[rows][:, 1:], x[:, None]], 1)
        return {"y": y, "state": state}
    per = case["channels"] // case["groups"]
    step = torch.logaddexp(s["dt"].double() + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    h = torch.exp(torch.einsum("tc,cn->tcn", step, s["a"].double())) * state[rows]
    h = h + torch.einsum("tc,tcn->tcn", step * x, s["b"].double().repeat_interleave(per, 1))
    y = torch.einsum("tcn,tcn->tc", h, s["c"].double().repeat_interleave(per, 1)) + s["d"].double() * x
    if case["gate"]:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    state[rows] = h
    return {"y": y, "state": state}


def _exact_norm(s):
    x = s["x"].double()
    ch = x.shape[1]
    mean = x.sum(1) / ch
    off = x - mean[:, None]
    rstd = ((off * off).sum(1) / ch + 1e-5) ** -0.5
    hat = off * rstd[:, None]
    w = s["weight"].double()
    out = {"y": hat * w + s["bias"].double(), "mean": mean, "rstd": rstd}
    if s["case"]["op"] == "norm_train":
        dy = s["dy"].double()
        along = (dy * w * hat).sum(1, keepdim=True)
        out["dx"] = rstd[:, None] / ch * (ch * dy * w - (dy * w).sum(1, keepdim=True) - hat * along)
        out["dweight"], out["dbias"] = (dy * hat).sum(0), dy.sum(0)
    return out


def exact(case, seed):
    op = case["op"]
    if op.startswith("scan") and op != "scan_token" and case["tokens"] * case["channels"] * case["states"] > 12e8:
        return None
    s = prepare(case, seed)
    if op.startswith("norm"):
        return _exact_norm(s)
    if op.endswith("_token"):
        return _exact_token(s)
    return _exact_conv(s) if op.startswith("conv") else _exact_scan(s)
