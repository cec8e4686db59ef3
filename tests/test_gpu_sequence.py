"""The sequence operators on the GPU against their formulas in 64 bits: the short
causal convolution, the selective scan and layer norm, with gradients and single
tokens; masks of sequences, states, slots, strides, streams and graphs."""
import pytest
import torch

import sequence_oracle as R
from sparsl_b200 import OpError

pytestmark = pytest.mark.gpu
F64 = torch.float64
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAN = float("nan")


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _rows(g, tokens, ch, dtype, wide=0, scale=1.0):
    """A token array on the GPU: contiguous, or a column range of a wider one."""
    v = (torch.randn(tokens, ch + wide, generator=g) * scale).to(dtype).cuda()
    return v[:, wide:]


def _up(t):
    return None if t is None else t.detach().cpu().to(F64)


def _stream():
    return torch.cuda.current_stream()


def _room(n):
    return torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")


class Scan:
    """A scan's inputs, its run on the GPU, and the oracle's."""

    def __init__(self, lens, ch, ns, groups=1, dtype=torch.float32, gate=True, skip=True, bias=True, softplus=True, state=False,
                 ragged=True, lead=0, tail=0, wide=0, seed=1):
        g = _gen(seed)
        self.lens, self.ch, self.ns, self.groups, self.dtype, self.softplus = lens, ch, ns, groups, dtype, softplus
        self.used = sum(lens)
        self.lead, self.tokens = lead, lead + self.used + tail
        self.ptr = torch.tensor(R.lengths_to_ptr(lens, lead), dtype=torch.int32).cuda() if ragged else None
        self.x = _rows(g, self.tokens, ch, dtype, wide)
        self.dt = _rows(g, self.tokens, ch, dtype, wide, 0.5)
        self.z = _rows(g, self.tokens, ch, dtype, wide) if gate else None
        self.a = (-torch.arange(1, ns + 1, dtype=torch.float32) * torch.exp(0.2 * torch.randn(ch, ns, generator=g))).cuda()
        rows = torch.randn(self.tokens, 5 + 2 * groups * ns, generator=g).to(dtype).cuda()
        self.b, self.c = (rows[:, k:k + groups * ns].unflatten(1, (groups, ns)) for k in (5, 5 + groups * ns))
        self.d = torch.randn(ch, generator=g).cuda() if skip else None
        step = torch.exp(torch.rand(ch, generator=g) * 4.6 - 6.9)
        self.bias = torch.log(torch.expm1(step)).cuda() if bias else None
        if not softplus:
            self.dt = self.dt.abs() * 0.1
            self.bias = step.cuda() if bias else None
        self.state = torch.randn(len(lens), ch, ns, generator=g).cuda() if state else None
        self.dy = _rows(g, self.tokens, ch, dtype, wide)
        self.dfinal = torch.randn(len(lens), ch, ns, generator=g).cuda() if state else None
        for t in (self.x, self.dt, self.z, self.b, self.c, self.dy):  # rows of no sequence are never read
            if t is not None:
                t[:lead] = NAN
                t[lead + self.used:] = NAN

    def seqs(self):
        return {"seq_ptr": self.ptr} if self.ptr is not None else {"n_seq": len(self.lens)}

    def live(self, t):
        return t[self.lead:self.lead + self.used]

    def forward(self, dev, marks=None, state=None, final=None, stream=None, **more):
        y = torch.full((self.tokens, self.ch), 7.0, dtype=self.dtype, device="cuda")
        room = _room(dev.selective_scan_workspace(self.tokens, self.ch, self.ns, len(self.lens), self.groups))
        dev.selective_scan_device(self.x, self.dt, self.a, self.b, self.c, y, room, d=self.d, z=self.z, dt_bias=self.bias,
                                  softplus=self.softplus, **self.seqs(), state=state, final_state=final, checkpoints=marks,
                                  stream=stream or _stream(), **more)
        return y

    def backward(self, dev, marks, stream=None):
        n = len(self.lens)
        out = {"dx": torch.full_like(self.x, 7.0), "ddt": torch.full_like(self.x, 7.0), "da": torch.full_like(self.a, NAN),
               "db": torch.full(self.b.shape, 7.0, dtype=self.dtype, device="cuda"),
               "dc": torch.full(self.b.shape, 7.0, dtype=self.dtype, device="cuda"),
               "dd": torch.full((self.ch,), NAN, device="cuda") if self.d is not None else None,
               "dz": torch.full_like(self.x, 7.0) if self.z is not None else None,
               "ddt_bias": torch.full((self.ch,), NAN, device="cuda") if self.bias is not None else None,
               "dstate": torch.full((n, self.ch, self.ns), NAN, device="cuda") if self.state is not None else None}
        room = _room(dev.selective_scan_backward_workspace(self.tokens, self.ch, self.ns, n, self.groups))
        room.fill_(255)  # NaNs: nothing may be read before it is written
        dev.selective_scan_backward_device(self.dy, self.x, self.dt, self.a, self.b, self.c, marks, out["dx"], out["ddt"],
                                           out["da"], out["db"], out["dc"], room, d=self.d, dd=out["dd"], z=self.z,
                                           dz=out["dz"], dt_bias=self.bias, ddt_bias=out["ddt_bias"],
                                           softplus=self.softplus, **self.seqs(), state=self.state,
                                           dstate=out["dstate"], dfinal_state=self.dfinal, stream=stream or _stream())
        return {k: v for k, v in out.items() if v is not None}

    def marks(self, dev):
        m = _room(dev.selective_scan_checkpoints(self.tokens, self.ch, self.ns))
        m.fill_(255)
        return m

    def oracle(self, start=None, backward=False):
        """{name: (value, magnitude)}, and the bound's factor."""
        both = []
        for magnitude in (False, True):
            leaf = {k: _up(self.live(getattr(self, k))) for k in ("x", "dt", "b", "c")}
            leaf.update(a=_up(self.a), d=_up(self.d), dt_bias=_up(self.bias), z=None if self.z is None else _up(self.live(self.z)),
                        start=_up(start))
            if magnitude:  # derivatives by absolute values
                for k in ("x", "b", "c", "d", "start"):
                    leaf[k] = None if leaf[k] is None else leaf[k].abs()
            if backward:
                for v in leaf.values():
                    if v is not None:
                        v.requires_grad_()
            y, final = R.scan(softplus=self.softplus, lens=self.lens, magnitude=magnitude, **leaf)
            out = {"y": y.detach(), "final": final.detach()}
            if backward:
                dy = _up(self.live(self.dy))
                loss = (y * (dy.abs() if magnitude else dy)).sum()
                if self.dfinal is not None:
                    df = _up(self.dfinal)
                    loss = loss + (final * (df.abs() if magnitude else df)).sum()
                names = {"x": "dx", "dt": "ddt", "a": "da", "b": "db", "c": "dc", "d": "dd", "z": "dz", "dt_bias": "ddt_bias",
                         "start": "dstate"}
                want = [k for k in names if leaf[k] is not None]
                grads = torch.autograd.grad(loss, [leaf[k] for k in want], allow_unused=True)
                for k, v in zip(want, grads):
                    out[names[k]] = torch.zeros_like(leaf[k]) if v is None else v
            both.append(out)
        k = R.scan_bound(_up(self.live(self.dt)), _up(self.a), _up(self.bias), self.softplus, self.lens, self.used, self.ch, backward)
        return {n: (both[0][n], both[1][n]) for n in both[0]}, k

    def untouched(self, t):
        """Rows in front of the first sequence and behind the last stay as they were."""
        assert (t[:self.lead] == 7).all() and (t[self.lead + self.used:] == 7).all()


SHAPES = [
    # lens, channels, states, groups, more
    dict(lens=[1], ch=1, ns=1),
    dict(lens=[5], ch=33, ns=16, ragged=False),
    dict(lens=[0], ch=8, ns=4),
    dict(lens=[], ch=8, ns=4),
    dict(lens=[31, 0, 1, 64, 0, 0, 33], ch=70, ns=16, lead=3, tail=4, wide=70),
    dict(lens=[64, 64, 64], ch=64, ns=16, ragged=False),
    dict(lens=[100, 100], ch=129, ns=11, groups=3, ragged=False),
    dict(lens=[290, 7], ch=24, ns=16, groups=2, tail=1),
    dict(lens=[150], ch=40, ns=8, ragged=False, gate=False),
    dict(lens=[3, 130], ch=20, ns=32, groups=4, skip=False, bias=False),
    dict(lens=[130, 2], ch=10, ns=64, softplus=False),
    dict(lens=[70], ch=12, ns=37, gate=False, skip=False),
    dict(lens=[96, 96], ch=260, ns=5, ragged=False),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(v) for v in s.values()))
def test_scan_forward(cuda_device, shape, state, dtype):
    s = Scan(dtype=dtype, state=state, **shape)
    final = torch.full_like(s.state, NAN) if state else None
    want, k = s.oracle(s.state)
    y = s.forward(cuda_device, state=s.state, final=final)
    R.check(s.live(y), *want["y"], k, "y")
    s.untouched(y)
    if state:
        R.check(final, *want["final"], k, "final")
        pool = s.state.clone()
        y2 = s.forward(cuda_device, state=pool, final=pool)  # in place
        assert torch.equal(y, y2) and torch.equal(final, pool)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(v) for v in s.values()))
def test_scan_backward(cuda_device, shape, state, dtype):
    s = Scan(dtype=dtype, state=state, **shape)
    marks = s.marks(cuda_device)
    want, k = s.oracle(s.state, backward=True)
    y = s.forward(cuda_device, marks=marks, state=s.state)
    R.check(s.live(y), *want["y"], k, "y")
    got = s.backward(cuda_device, marks)
    for name, v in got.items():
        token = name in ("dx", "ddt", "db", "dc", "dz")
        R.check(s.live(v) if token else v, *want[name], k, name)
        if token:
            s.untouched(v)
    again = s.backward(cuda_device, marks)
    for name, v in got.items():
        assert torch.equal(v, again[name]), name


def test_scan_slots_and_resume(cuda_device):
    """Rows of a pool by slot: some sequences start anew, some have no row; the rest of the pool stays."""
    s = Scan([40, 100, 0, 3, 0, 70, 9], 50, 16, tail=2)
    g = _gen(5)
    pool = torch.randn(11, 50, 16, generator=g).cuda()
    slots = torch.tensor([4, 0, 10, -1, 7, 2, 99], dtype=torch.int32).cuda()  # 99: outside, none
    resume = torch.tensor([1, 0, 1, 1, 0, 1, 1], dtype=torch.uint8).cuda()
    start = torch.zeros(7, 50, 16)
    for i, (r, f) in enumerate(zip(slots.tolist(), resume.tolist())):
        if 0 <= r < 11 and f:
            start[i] = pool[r].cpu()
    want, k = s.oracle(start)
    before = pool.clone()
    y = s.forward(cuda_device, state=pool, final=pool, slots=slots, resume=resume)
    R.check(s.live(y), *want["y"], k, "y")
    for i, r in enumerate(slots.tolist()):
        if 0 <= r < 11:
            R.check(pool[r], want["final"][0][i], want["final"][1][i], k, f"pool row {r}")
    rest = [r for r in range(11) if r not in slots.tolist()]
    assert torch.equal(pool[rest], before[rest])
    assert torch.equal(pool[10], before[10]) and (pool[7] == 0).all()  # empty: kept, or begun anew


@pytest.mark.parametrize("ns", [1, 4, 7, 16, 30, 64])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scan_tokens_one_by_one(cuda_device, ns, dtype):
    """Steps through a pool give what the prompt gives."""
    n, ch, groups, steps = 5, 36, 2, 6
    g = _gen(ns)
    s = Scan([steps] * n, ch, ns, groups, dtype, state=True, ragged=False, wide=36)
    want, k = s.oracle(s.state)
    pool = torch.randn(9, ch, ns, generator=g).cuda()
    slots = torch.tensor([8, 1, -1, 0, 5], dtype=torch.int32).cuda()
    for i, r in enumerate(slots.tolist()):
        if r >= 0:
            pool[r] = s.state[i]
    before = pool.clone()
    pick = lambda t, k: t.unflatten(0, (n, steps))[:, k]  # noqa: E731
    for k_ in range(steps):
        y = torch.full((n, ch), 7.0, dtype=dtype, device="cuda")
        cuda_device.selective_scan_step_device(pick(s.x, k_), pick(s.dt, k_), s.a, pick(s.b, k_), pick(s.c, k_), y, pool, d=s.d,
                                               z=pick(s.z, k_), dt_bias=s.bias, softplus=True, slots=slots, stream=_stream())
        for i, r in enumerate(slots.tolist()):
            if r < 0:
                assert (y[i] == 7).all()
                continue
            R.check(y[i], want["y"][0].unflatten(0, (n, steps))[i, k_], want["y"][1].unflatten(0, (n, steps))[i, k_], k, "y")
    for i, r in enumerate(slots.tolist()):
        if r >= 0:
            R.check(pool[r], want["final"][0][i], want["final"][1][i], k, "state")
    rest = [r for r in range(9) if r not in slots.tolist()]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("ns", [16, 8, 5, 20, 40, 64])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scan_tokens_of_many_sequences(cuda_device, ns, dtype):
    """A batch large enough for the kernel that takes several sequences a block; some have no state."""
    n, ch = 603, 514
    s = Scan([1] * n, ch, ns, 2, dtype, state=True, ragged=False)
    slots = torch.randperm(n + 7, generator=_gen(ns))[:n].to(torch.int32)
    slots[[3, 4, 100, 602]] = -1
    rows = slots.tolist()
    pool = torch.full((n + 7, ch, ns), 3.0, device="cuda")
    live = torch.tensor([i for i, r in enumerate(rows) if r >= 0])
    pool[slots[live].long()] = s.state[live.cuda()]
    before = pool.clone()
    y = torch.full((n, ch), 7.0, dtype=dtype, device="cuda")
    cuda_device.selective_scan_step_device(s.x, s.dt, s.a, s.b, s.c, y, pool, d=s.d, z=s.z, dt_bias=s.bias, softplus=True,
                                           slots=slots.cuda(), stream=_stream())
    want, k = s.oracle(s.state)
    R.check(y[live.cuda()], want["y"][0][live], want["y"][1][live], k, "y")
    R.check(pool[slots[live].long()], want["final"][0][live], want["final"][1][live], k, "state")
    assert (y[[3, 4, 100, 602]] == 7).all()
    rest = [r for r in range(n + 7) if r not in rows]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("shape", [dict(lens=[1] * 333, ch=40, ns=16, tail=3), dict(lens=[2, 1, 3] * 60, ch=17, ns=8, lead=9),
                                   dict(lens=[64] * 40, ch=260, ns=16, ragged=False), dict(lens=[32] * 9, ch=1200, ns=4, ragged=False),
                                   dict(lens=[96] * 12, ch=384, ns=32, ragged=False, groups=2)], ids=str)
def test_scan_many_sequences(cuda_device, shape):
    s = Scan(state=True, dtype=torch.bfloat16, **shape)
    marks = s.marks(cuda_device)
    want, k = s.oracle(s.state, backward=True)
    final = torch.full_like(s.state, NAN)
    y = s.forward(cuda_device, marks=marks, state=s.state, final=final)
    R.check(s.live(y), *want["y"], k, "y")
    R.check(final, *want["final"], k, "final")
    s.untouched(y)
    for name, v in s.backward(cuda_device, marks).items():
        R.check(s.live(v) if name in ("dx", "ddt", "db", "dc", "dz") else v, *want[name], k, name)


def _layout(tokens, ch, ns, n_seq, groups, ragged, backward):
    """(lanes a channel, chunks, their tokens, states handed on, lanes of the pass that computes those)."""
    import ctypes

    from sparsl_b200 import _lib

    out = (ctypes.c_uint64 * 5)()
    assert _lib.load().sparsl_selective_scan_test_layout(tokens, ch, ns, n_seq, groups, ragged, backward, out) == 0
    return list(out)


def _part(s, seqs, groups):
    """Some sequences and groups of a scan, as its oracle takes them: what they give does not depend on the others."""
    import copy

    per, at = s.ch // s.groups, R.lengths_to_ptr(s.lens)
    rows = torch.cat([torch.arange(at[i], at[i + 1]) for i in seqs]).cuda()
    cols = torch.cat([torch.arange(g * per, (g + 1) * per) for g in groups]).cuda()
    p = copy.copy(s)
    p.lens, p.ch, p.groups, p.lead = [s.lens[i] for i in seqs], len(cols), len(groups), 0
    p.used = p.tokens = len(rows)
    for k in ("x", "dt", "z", "dy"):
        setattr(p, k, None if getattr(s, k) is None else s.live(getattr(s, k))[rows][:, cols])
    p.b, p.c = (s.live(v)[rows][:, groups] for v in (s.b, s.c))
    p.a, p.d, p.bias = (None if v is None else v[cols] for v in (s.a, s.d, s.bias))
    p.state, p.dfinal = (None if v is None else v[list(seqs)][:, cols] for v in (s.state, s.dfinal))
    return p, rows, cols


# Sizes at which a scan takes the layouts that large inputs take: one of few lanes a channel with states handed on, and whole
# sequences with two lanes.  `ahead` is the layout of the prompt, `back` of the gradients: lanes, handed on, the chunk pass's lanes.
MANY = [70, 1300, 0, 1, 64, 129, 3]
LARGE = [
    dict(lens=MANY, ns=16, dtype=torch.bfloat16, ahead=(1, 1, 1), back=(2, 1, 4)),
    dict(lens=MANY, ns=16, dtype=torch.float16, ahead=(1, 1, 1), back=(2, 1, 4)),
    dict(lens=MANY, ns=11, dtype=torch.float32, ahead=(1, 1, 1), back=(2, 1, 4)),
    dict(lens=MANY, ns=8, dtype=torch.bfloat16, ahead=(1, 1, 1), back=(1, 1, 2)),
    dict(lens=MANY, ns=5, dtype=torch.float32, ahead=(1, 1, 1), back=(1, 1, 2), gate=False),
    dict(lens=MANY, ns=32, dtype=torch.bfloat16, ahead=(2, 1, 2), back=(4, 1, 4)),
    dict(lens=MANY, ns=23, dtype=torch.float16, ahead=(2, 1, 2), back=(4, 1, 4), gate=False),
    dict(lens=MANY, ns=64, dtype=torch.bfloat16, ahead=(4, 1, 4), back=(8, 1, 4)),
    dict(lens=[96] * 8, ns=16, dtype=torch.bfloat16, ahead=(2, 0, 0), back=(2, 0, 0), ragged=False, ch=2048, groups=16),
    dict(lens=[96] * 8, ns=13, dtype=torch.float32, ahead=(2, 0, 0), back=(2, 0, 0), ragged=False, ch=2048, groups=16),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"{c['ns']}-{str(c['dtype'])[6:]}-{'-'.join(map(str, c['ahead'] + c['back']))}")
def test_scan_layouts_of_large_inputs(cuda_device, case):
    case = dict(case)
    ahead, back = case.pop("ahead"), case.pop("back")
    ragged = case.get("ragged", True)
    case = {"ch": 4096, "groups": 32, "lead": 2 * ragged, "tail": 5 * ragged, **case}
    s = Scan(state=True, **case)
    n = len(s.lens)
    for want, b in ((ahead, False), (back, True)):
        lanes, chunks, _, carry, first = _layout(s.tokens, s.ch, s.ns, n, s.groups, ragged, b)
        assert (lanes, carry, first) == want and (chunks > 1 or not carry)
    marks = s.marks(cuda_device)
    final = torch.full_like(s.state, NAN)
    y = s.forward(cuda_device, marks=marks, state=s.state, final=final)
    got = s.backward(cuda_device, marks)
    # In place, in a pool by slot; one sequence begins anew, one keeps no state.
    slots = torch.randperm(n + 3, generator=_gen(4))[:n].to(torch.int32)
    slots[0] = -1
    resume = torch.ones(n, dtype=torch.uint8)
    resume[1] = 0
    pool = torch.full((n + 3, s.ch, s.ns), 3.0, device="cuda")
    pool[slots[1:].long().cuda()] = s.state[1:]
    y2 = s.forward(cuda_device, state=pool, final=pool, slots=slots.cuda(), resume=resume.cuda())
    s.untouched(y)
    s.untouched(y2)
    groups = [0, s.groups // 2, s.groups - 1]
    p, rows, cols = _part(s, range(n), groups)
    want, k = p.oracle(p.state, backward=True)
    pick = lambda v: s.live(v)[:, cols]  # noqa: E731
    R.check(pick(y), *want["y"], k, "y")
    R.check(final[:, cols], *want["final"], k, "final")
    for name, v in got.items():
        if name in ("db", "dc"):
            v = s.live(v)[:, groups]
        elif name in ("dx", "ddt", "dz"):
            s.untouched(v)
            v = pick(v)
        else:
            v = v[:, cols] if name == "dstate" else v[cols]
        R.check(v, *want[name], k, name)
    start = p.state.clone()
    start[:2] = 0
    want, k = p.oracle(start)
    R.check(pick(y2), *want["y"], k, "y, in place")
    kept = slots[1:].long()
    R.check(pool[kept.cuda()][:, cols], *(v[1:] for v in want["final"]), k, "pool")
    rest = [r for r in range(n + 3) if r not in slots.tolist()]
    assert (pool[rest] == 3).all()


def test_scan_of_very_many_chunks(cuda_device):
    """One tile of channels over hundreds of chunks: the first, the last and a long sequence against the formulas."""
    lens = [900, 3, 1, 40] + [1300] * 21 + [300, 64]
    s = Scan(lens, 64, 16, dtype=torch.bfloat16, state=True)
    assert _layout(s.tokens, 64, 16, len(lens), 1, True, False)[3:] == [1, 1]
    lanes, chunks, _, carry, first = _layout(s.tokens, 64, 16, len(lens), 1, True, True)
    assert (lanes, carry, first) == (2, 1, 4) and chunks >= 444
    marks = s.marks(cuda_device)
    final = torch.full_like(s.state, NAN)
    y = s.forward(cuda_device, marks=marks, state=s.state, final=final)
    got = s.backward(cuda_device, marks)
    seqs = [0, 3, 14, len(lens) - 1]
    p, rows, _ = _part(s, seqs, [0])
    want, k = p.oracle(p.state, backward=True)
    R.check(y[rows], *want["y"], k, "y")
    R.check(final[seqs], *want["final"], k, "final")
    for name in ("dx", "ddt", "db", "dc", "dz"):
        R.check(got[name][rows], *want[name], k, name)
    R.check(got["dstate"][seqs], *want["dstate"], k, "dstate")


def test_scan_infinite_and_nan_stay_in_their_sequence(cuda_device):
    s = Scan([50, 40, 60], 20, 11)
    clean = s.forward(cuda_device)
    s.x[60] = float("inf")
    s.dt[55, 3] = NAN
    y = s.forward(cuda_device)
    assert torch.equal(y[:50], clean[:50]) and torch.equal(y[90:], clean[90:])
    assert not torch.isfinite(y[60:90]).all() and torch.isnan(y[55:90, 3]).all()
    assert torch.equal(y[50:55], clean[50:55])


@pytest.mark.parametrize("start,rate", [(1e-30, 1.45), (0.0, 2.0), (1e30, -1.45)])
def test_states_across_chunks_that_grow_or_fade_past_a_float(cuda_device, start, rate):
    """A chunk's whole decay may leave f32's range where no state does: exp(+-93) of a state of 1e-+30, exp(128) of none."""
    t, ch, ns, chunk = 192, 8, 4, 64
    x = torch.zeros(t, ch, device="cuda")
    x[2 * chunk:] = 1
    dt = torch.zeros(t, ch, device="cuda")
    dt[chunk:2 * chunk] = 1
    dt[2 * chunk:] = 2.0 ** -10
    a = torch.full((ch, ns), rate, device="cuda")
    b, c = torch.full((t, ns), 0.0 if start else 1.0, device="cuda"), torch.ones(t, ns, device="cuda")
    state = torch.full((1, ch, ns), start, device="cuda")
    y, final = torch.zeros_like(x), torch.zeros_like(state)
    assert cuda_device.selective_scan_workspace(t, ch, ns, 1, 1) > 0  # chunks
    room = _room(cuda_device.selective_scan_workspace(t, ch, ns, 1, 1))
    ptr = torch.tensor([0, t], dtype=torch.int32).cuda()
    cuda_device.selective_scan_device(x, dt, a, b, c, y, room, seq_ptr=ptr, state=state, final_state=final, stream=_stream())
    leaf = [_up(v) for v in (x, dt, a, b[:, None], c[:, None])]
    want, last = R.scan(*leaf, None, None, None, False, [t], _up(state))
    most, most_last = R.scan(*leaf, None, None, None, False, [t], _up(state), magnitude=True)
    k = R.scan_bound(_up(dt), _up(a), None, False, [t], t, ch)
    R.check(y, want, most, k, "y")
    R.check(final, last, most_last, k, "final")


@pytest.mark.parametrize("chunked", [False, True])
def test_scan_without_a_skip_keeps_infinities(cuda_device, chunked):
    """Without d, an infinite x gives what the states give, and an infinite gradient what they take: not 0 times infinity."""
    inf = float("inf")
    t, ch = (300, 3) if chunked else (40, 3)
    x = torch.ones(t, ch, device="cuda")
    dt, a = torch.ones(t, ch, device="cuda"), torch.full((ch, 8), -0.5, device="cuda")
    b, c = torch.ones(t, 8, device="cuda"), torch.ones(t, 8, device="cuda")
    x[t - 3, 1] = inf
    y = torch.zeros_like(x)
    room = _room(max(cuda_device.selective_scan_workspace(t, ch, 8), cuda_device.selective_scan_backward_workspace(t, ch, 8)))
    marks = _room(cuda_device.selective_scan_checkpoints(t, ch, 8))
    for ptr in (None, torch.tensor([0, t - 1], dtype=torch.int32).cuda()):  # whole batches, and an end inside one
        cuda_device.selective_scan_device(x, dt, a, b, c, y, room, seq_ptr=ptr, checkpoints=marks, stream=_stream())
        assert (y[t - 3:t - 1, 1] == inf).all() and torch.isfinite(y[:, [0, 2]]).all() and torch.isfinite(y[:t - 3]).all()
    state = torch.zeros(1, ch, 8, device="cuda")
    y1 = torch.zeros(1, ch, device="cuda")
    cuda_device.selective_scan_step_device(x[t - 3:t - 2], dt[:1], a, b[:1], c[:1], y1, state, stream=_stream())
    assert y1[0, 1] == inf
    n = 2400
    ym, xm = torch.zeros(n, 512, device="cuda"), torch.ones(n, 512, device="cuda")
    xm[5, 7] = inf
    am, one = torch.full((512, 8), -0.5, device="cuda"), torch.ones(n, 8, device="cuda")
    cuda_device.selective_scan_step_device(xm, torch.ones_like(xm), am, one, one, ym, torch.zeros(n, 512, 8, device="cuda"),
                                           stream=_stream())
    assert ym[5, 7] == inf and torch.isfinite(ym).sum() == n * 512 - 1
    x[t - 3, 1] = 1
    dy = torch.ones_like(x)
    dy[t - 3, 1] = inf
    dx, ddt, da, db, dc = (torch.zeros_like(k) for k in (x, dt, a, b, c))
    z = torch.ones_like(x)
    cuda_device.selective_scan_device(x, dt, a, b, c, y, room, z=z, checkpoints=marks, stream=_stream())
    dz = torch.zeros_like(x)
    cuda_device.selective_scan_backward_device(dy, x, dt, a, b, c, marks, dx, ddt, da, db, dc, room, z=z, dz=dz, stream=_stream())
    assert (dx[:t - 2, 1] == inf).all() and torch.isfinite(dx[t - 2:]).all() and torch.isfinite(dx[:, [0, 2]]).all()


@pytest.mark.parametrize("ns,ragged", [(16, True), (16, False), (5, False)])
def test_scan_long_memory_is_not_biased(cuda_device, ns, ragged):
    """States that only fade, over 1024 tokens: their mean relative error stays below 1e-8 a token, half of what the special
    function unit's powers of two alone are low by, and 1e-6 for the mean of the roundings; with a step of zero the bits stay."""
    t, ch = 1024, 64
    g = _gen(3)
    # s a in (-0.06, 0), so that the states end above exp(-62) of their start.
    dt, a = torch.rand(t, ch, generator=g) * 0.06, -torch.rand(ch, ns, generator=g)
    state = 1 + torch.rand(1, ch, ns, generator=g)
    final = torch.zeros(1, ch, ns, device="cuda")
    zero = torch.zeros(t, ch, device="cuda")
    room = _room(cuda_device.selective_scan_workspace(t, ch, ns))
    ptr = torch.tensor([0, t], dtype=torch.int32).cuda() if ragged else None

    def run(dt):
        cuda_device.selective_scan_device(zero, dt, a.cuda(), torch.zeros(t, ns, device="cuda"), torch.zeros(t, ns, device="cuda"),
                                          torch.zeros_like(zero), room, seq_ptr=ptr, state=state.cuda(), final_state=final,
                                          stream=_stream())
        return _up(final[0])

    want = _up(state[0]) * torch.exp(_up(dt).sum(0)[:, None] * _up(a))
    off = run(dt.cuda()) / want - 1
    assert abs(float(off.mean())) < t * 1e-8 + 1e-6, float(off.mean())
    assert torch.equal(run(zero), _up(state[0]))
    pool = state.cuda()  # token by token
    row = torch.zeros(1, ns, device="cuda")
    steps = dt.cuda()
    for k in range(t):
        cuda_device.selective_scan_step_device(zero[:1], steps[k:k + 1], a.cuda(), row, row, torch.zeros(1, ch, device="cuda"), pool,
                                               stream=_stream())
    off = _up(pool[0]) / want - 1
    assert abs(float(off.mean())) < t * 1e-8 + 1e-6, float(off.mean())


def test_scan_far_states(cuda_device):
    """A pool whose rows lie past 2^32 bytes and 2^31 values."""
    ch, ns, rows = 2048, 16, 70000
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("the pool does not fit this GPU")
    s = Scan([40], ch, ns, state=True)
    want, k = s.oracle(s.state)
    pool = torch.empty(rows, ch, ns, device="cuda")
    slots = torch.tensor([rows - 1], dtype=torch.int32).cuda()
    pool[rows - 1] = s.state[0]
    y = s.forward(cuda_device, state=pool, final=pool, slots=slots)
    R.check(y, *want["y"], k, "y")
    R.check(pool[rows - 1], want["final"][0][0], want["final"][1][0], k, "final")
    pool[rows - 1] = s.state[0]
    yt = torch.empty(1, ch, device="cuda")
    cuda_device.selective_scan_step_device(s.x[:1], s.dt[:1], s.a, s.b[:1], s.c[:1], yt, pool, d=s.d, z=s.z[:1], dt_bias=s.bias,
                                           softplus=True, slots=slots, stream=_stream())
    R.check(yt, want["y"][0][:1], want["y"][1][:1], k, "step")


def test_kept_states_and_workspaces_past_half_a_gigabyte(cuda_device):
    """129 equal sequences whose kept states and workspace pass 2^29 bytes give what one gives, bit for bit."""
    dev, st = cuda_device, _stream()
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("the arrays do not fit this GPU")
    n, length, ch, ns, dtype = 129, 64, 2048, 64, torch.bfloat16
    one = Scan([length], ch, ns, dtype=dtype, ragged=False)
    names = ("x", "dt", "z", "b", "c", "dy")
    rows = {k: getattr(one, k).repeat(n, *([1] * (getattr(one, k).dim() - 1))) for k in names}
    t = n * length
    assert dev.selective_scan_checkpoints(t, ch, ns) >= 1 << 29
    assert dev.selective_scan_backward_workspace(t, ch, ns, n) >= 1 << 29

    def both(x, dt, z, b, c, dy, n):
        t = x.shape[0]
        y, dx, ddt, dz = (torch.zeros_like(x) for _ in range(4))
        db, dc, da, dd, dbias = (torch.zeros(k.shape, dtype=k.dtype, device="cuda") for k in (b, c, one.a, one.d, one.bias))
        marks = _room(dev.selective_scan_checkpoints(t, ch, ns))
        room = _room(max(dev.selective_scan_workspace(t, ch, ns, n), dev.selective_scan_backward_workspace(t, ch, ns, n)))
        dev.selective_scan_device(x, dt, one.a, b, c, y, room, d=one.d, z=z, dt_bias=one.bias, softplus=True, n_seq=n,
                                  checkpoints=marks, stream=st)
        dev.selective_scan_backward_device(dy, x, dt, one.a, b, c, marks, dx, ddt, da, db, dc, room, d=one.d, dd=dd, z=z, dz=dz,
                                           dt_bias=one.bias, ddt_bias=dbias, softplus=True, n_seq=n, stream=st)
        return (y, dx, ddt, dz, db, dc), (da, dd, dbias)

    small, small_sums = both(*(getattr(one, k).contiguous() for k in names), 1)
    large, sums = both(*(rows[k] for k in names), n)
    for p, q in zip(small, large):
        assert torch.equal(q.unflatten(0, (n, length)), p.expand(n, *p.shape))
    for p, q in zip(small_sums, sums):  # n equal terms, each addition rounded once
        assert ((q.double() - n * p.double()).abs() <= n * 2.0 ** -24 * n * p.double().abs()).all()


def test_rows_of_the_scan_lie_within_their_reach(cuda_device):
    """The scan counts a row's bytes in 31 bits: longer strides are refused."""
    s = Scan([2], 4, 4)
    far = torch.empty((1 << 29) + 8, dtype=torch.bfloat16, device="cuda").as_strided((2, 4), (1 << 29, 1))
    args = [v.to(torch.bfloat16) for v in (s.x, s.dt)]
    bc = [v.to(torch.bfloat16).contiguous() for v in (s.b, s.c)]
    assert "stride" in _refused("Length", cuda_device.selective_scan_device, far, args[1], s.a, *bc, torch.zeros_like(args[0]), None,
                                stream=_stream())


def test_scan_gradients_of_very_many_groups(cuda_device):
    """The partial sums of eight tokens' B and C pass 2^32 values: each group gives what one alone gives, bit for bit."""
    dev, st = cuda_device, _stream()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("the groups do not fit this GPU")
    n, ns, t = 4_800_000, 64, 8
    one = Scan([t], 1, ns, dtype=torch.bfloat16, gate=False, skip=False, bias=False, softplus=False, ragged=False)

    def grads(n):
        x, dt, dy = (v.expand(t, n).contiguous() for v in (one.x, one.dt, one.dy))
        a = one.a.expand(n, ns).contiguous()
        b, c = (v.expand(t, n, ns).contiguous() for v in (one.b, one.c))
        y, dx, ddt, da, db, dc = (torch.zeros_like(v) for v in (x, x, x, a, b, c))
        marks = _room(dev.selective_scan_checkpoints(t, n, ns))
        room = _room(dev.selective_scan_backward_workspace(t, n, ns, 1, n))
        dev.selective_scan_device(x, dt, a, b, c, y, None, checkpoints=marks, stream=st)
        dev.selective_scan_backward_device(dy, x, dt, a, b, c, marks, dx, ddt, da, db, dc, room, stream=st)
        return y, dx, ddt, da[None], db, dc

    alone = grads(1)
    for p, q in zip(alone, grads(n)):
        assert (q == p.expand_as(q)).all()
    del q
    torch.cuda.empty_cache()  # 45 GB


# ---- the causal convolution ----------------------------------------------------------------------


class Conv:
    def __init__(self, lens, ch, width, dtype=torch.float32, bias=True, silu=True, state=False, ragged=True, lead=0, tail=0,
                 wide=0, params=None, seed=2):
        g = _gen(seed)
        self.lens, self.ch, self.width, self.dtype, self.silu = lens, ch, width, dtype, silu
        self.used = sum(lens)
        self.lead, self.tokens = lead, lead + self.used + tail
        self.ptr = torch.tensor(R.lengths_to_ptr(lens, lead), dtype=torch.int32).cuda() if ragged else None
        self.x, self.dy = _rows(g, self.tokens, ch, dtype, wide), _rows(g, self.tokens, ch, dtype, wide)
        params = params or torch.float32
        self.w = torch.randn(ch, width, generator=g).to(params).cuda()
        self.bias = torch.randn(ch, generator=g).to(params).cuda() if bias else None
        make = lambda: torch.randn(len(lens), width - 1, ch, generator=g).to(dtype).cuda()  # noqa: E731
        self.state, self.dfinal = (make(), make()) if state else (None, None)
        for t in (self.x, self.dy):
            t[:lead] = NAN
            t[lead + self.used:] = NAN

    seqs, live, untouched = Scan.seqs, Scan.live, Scan.untouched

    def forward(self, dev, state=None, final=None, stream=None, **more):
        y = torch.full((self.tokens, self.ch), 7.0, dtype=self.dtype, device="cuda")
        dev.causal_conv_device(self.x, self.w, y, bias=self.bias, silu=self.silu, **self.seqs(), state=state, final_state=final,
                               stream=stream or _stream(), **more)
        return y

    def backward(self, dev, stream=None):
        out = {"dx": torch.full_like(self.x, 7.0), "dw": torch.full((self.ch, self.width), NAN, device="cuda"),
               "dbias": torch.full((self.ch,), NAN, device="cuda") if self.bias is not None else None,
               "dstate": torch.full_like(self.state, NAN) if self.state is not None else None}
        room = _room(dev.causal_conv_backward_workspace(self.tokens, self.ch, self.width))
        room.fill_(255)
        dev.causal_conv_backward_device(self.dy, self.x, self.w, out["dx"], out["dw"], room, bias=self.bias, dbias=out["dbias"],
                                        silu=self.silu, **self.seqs(), state=self.state, dstate=out["dstate"],
                                        dfinal_state=self.dfinal, stream=stream or _stream())
        return {k: v for k, v in out.items() if v is not None}

    def oracle(self, start=None):
        both = []
        for magnitude in (False, True):
            leaf = {"x": _up(self.live(self.x)), "w": _up(self.w), "bias": _up(self.bias), "start": _up(start)}
            for k, v in leaf.items():
                if v is not None:
                    leaf[k] = (v.abs() if magnitude else v).requires_grad_()
            y, final = R.conv(leaf["x"], leaf["w"], leaf["bias"], self.silu, self.lens, leaf["start"], magnitude)
            out = {"y": y.detach(), "final": final.detach()}
            dy = _up(self.live(self.dy))
            loss = (y * (dy.abs() if magnitude else dy)).sum()
            if self.dfinal is not None:
                df = _up(self.dfinal)
                loss = loss + (final * (df.abs() if magnitude else df)).sum()
            want = [k for k in leaf if leaf[k] is not None]
            grads = torch.autograd.grad(loss, [leaf[k] for k in want], allow_unused=True)
            for k, v in zip(want, grads):
                out[{"x": "dx", "w": "dw", "bias": "dbias", "start": "dstate"}[k]] = torch.zeros_like(leaf[k]) if v is None else v
            both.append(out)
        return {n: (both[0][n], both[1][n]) for n in both[0]}


# The sums of a token: width + 1 terms, the gate's three roundings of 2^-22; the parameters' sums add the tokens' roundings.
CONV_K = 32 * 2.0 ** -24

CONVS = [
    dict(lens=[1], ch=1, width=2),
    dict(lens=[7], ch=24, width=4, ragged=False),
    dict(lens=[0], ch=8, width=3),
    dict(lens=[], ch=8, width=3),
    dict(lens=[31, 0, 1, 64, 0, 0, 33, 2, 1, 1], ch=70, width=4, lead=3, tail=5, wide=70),
    dict(lens=[32, 32, 32, 32], ch=64, width=4, ragged=False),
    dict(lens=[30, 1, 1, 2, 1, 62, 1, 3], ch=40, width=4, silu=False),
    dict(lens=[63, 66, 1, 130], ch=260, width=3, bias=False),
    dict(lens=[200], ch=516, width=2, ragged=False, wide=4),
    dict(lens=[95, 33], ch=1031, width=4),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", CONVS, ids=lambda s: "-".join(str(v) for v in s.values()))
def test_conv(cuda_device, shape, state, dtype):
    s = Conv(dtype=dtype, state=state, **shape)
    want = s.oracle(s.state)
    final = torch.full_like(s.state, NAN) if state else None
    y = s.forward(cuda_device, state=s.state, final=final)
    R.check(s.live(y), *want["y"], CONV_K, "y")
    s.untouched(y)
    if state:
        assert torch.equal(_up(final), want["final"][0])  # inputs, moved
        pool = s.state.clone()
        assert torch.equal(s.forward(cuda_device, state=pool, final=pool), y) and torch.equal(pool, final)
    got = s.backward(cuda_device)
    R.check(s.live(got["dx"]), *want["dx"], CONV_K, "dx")
    s.untouched(got["dx"])
    for name in ("dw", "dbias"):
        if name in got:
            R.check(got[name], *want[name], CONV_K + s.used * 2.0 ** -24, name)
    if state:
        R.check(got["dstate"], *want["dstate"], CONV_K, "dstate")
    again = s.backward(cuda_device)
    for name, v in got.items():
        assert torch.equal(v, again[name]), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_conv_params_in_the_tokens_type(cuda_device, dtype):
    s = Conv([20, 40], 48, 4, dtype, params=dtype)
    want = s.oracle()
    R.check(s.forward(cuda_device), *want["y"], CONV_K, "y")
    got = s.backward(cuda_device)
    R.check(got["dx"], *want["dx"], CONV_K, "dx")
    R.check(got["dw"], *want["dw"], CONV_K + 60 * 2.0 ** -24, "dw")


def test_conv_slots_and_resume(cuda_device):
    s = Conv([33, 0, 2, 64, 0, 1], 20, 4, torch.bfloat16, tail=1)
    g = _gen(8)
    pool = torch.randn(9, 3, 20, generator=g).to(torch.bfloat16).cuda()
    slots = torch.tensor([3, 8, 0, -5, 1, 6], dtype=torch.int32).cuda()
    resume = torch.tensor([0, 1, 1, 1, 0, 1], dtype=torch.uint8).cuda()
    start = torch.zeros(6, 3, 20, dtype=torch.bfloat16)
    for i, (r, f) in enumerate(zip(slots.tolist(), resume.tolist())):
        if r >= 0 and f:
            start[i] = pool[r].cpu()
    want = s.oracle(start)
    before = pool.clone()
    y = s.forward(cuda_device, state=pool, final=pool, slots=slots, resume=resume)
    R.check(s.live(y), *want["y"], CONV_K, "y")
    for i, r in enumerate(slots.tolist()):
        if r >= 0:
            assert torch.equal(_up(pool[r]), want["final"][0][i]), r
    rest = [r for r in range(9) if r not in slots.tolist()]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("ch", [1, 30, 1032])
def test_conv_tokens_one_by_one(cuda_device, ch, dtype, width):
    n, steps = 4, 6
    s = Conv([steps] * n, ch, width, dtype, state=True, ragged=False, wide=ch)
    want = s.oracle(s.state)
    g = _gen(1)
    pool = torch.randn(7, width - 1, ch, generator=g).to(dtype).cuda()
    slots = torch.tensor([6, -1, 0, 3], dtype=torch.int32).cuda()
    for i, r in enumerate(slots.tolist()):
        if r >= 0:
            pool[r] = s.state[i]
    before = pool.clone()
    for k in range(steps):
        y = torch.full((n, ch), 7.0, dtype=dtype, device="cuda")
        cuda_device.causal_conv_step_device(s.x.unflatten(0, (n, steps))[:, k], s.w, y, pool, bias=s.bias, silu=True, slots=slots,
                                            stream=_stream())
        for i, r in enumerate(slots.tolist()):
            if r < 0:
                assert (y[i] == 7).all()
            else:
                R.check(y[i], want["y"][0].unflatten(0, (n, steps))[i, k], want["y"][1].unflatten(0, (n, steps))[i, k], CONV_K, "y")
    for i, r in enumerate(slots.tolist()):
        if r >= 0:
            assert torch.equal(_up(pool[r]), want["final"][0][i])
    rest = [r for r in range(7) if r not in slots.tolist()]
    assert torch.equal(pool[rest], before[rest])


# ---- layer norm ------------------------------------------------------------------------------------

NORMS = [(1, 1), (3, 2), (5, 31), (2, 32), (7, 33), (1000, 100), (4, 1024), (3, 1030), (300, 520), (2, 4096), (700, 2048), (9, 5003),
         (400, 8192), (3, 8200), (2, 16384), (301, 12001), (2, 33000), (0, 64),
         (2400, 104), (2369, 520), (2371, 1032), (2370, 2048), (2368, 4000), (2380, 6144), (2369, 8192), (2400, 33)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,ch", NORMS)
def test_norm(cuda_device, rows, ch, dtype):
    g = _gen(rows * 7 + ch)
    wide = 8 if ch % 2 == 0 else 0
    x = _rows(g, rows, ch, dtype, wide) + torch.tensor(0.5, dtype=dtype, device="cuda")
    dy = _rows(g, rows, ch, dtype, wide)
    w, bias = torch.randn(ch, generator=g).cuda(), torch.randn(ch, generator=g).cuda()
    y, dx = torch.full_like(x, NAN), torch.full((rows, ch), NAN, dtype=dtype, device="cuda")
    mean, rstd = torch.full((rows,), NAN, device="cuda"), torch.full((rows,), NAN, device="cuda")
    dw, db = torch.full((ch,), NAN, device="cuda"), torch.full((ch,), NAN, device="cuda")
    cuda_device.layer_norm_device(x, y, weight=w, bias=bias, eps=1e-5, mean=mean, rstd=rstd, stream=_stream())
    room = _room(cuda_device.layer_norm_backward_workspace(rows, ch))
    room.fill_(255)
    args = (dy, x, mean, rstd, dx, room)
    cuda_device.layer_norm_backward_device(*args, weight=w, dweight=dw, dbias=db, stream=_stream())
    if rows == 0:
        assert (dw == 0).all() and (db == 0).all()
        return
    leaf = [_up(v).requires_grad_() for v in (x, w, bias)]
    wy, wm, wr = R.norm(*leaf, 1e-5)
    gx, gw, gb = torch.autograd.grad((wy * _up(dy)).sum(), leaf)
    # Row sums are trees of at most 32 serial terms and 10 levels (long rows: ch / 1024 terms): their relative error is
    # below k of the sum of absolute values, the deviations' below 2k of (|x - mean| + mean |x|), the variance's below 4k of
    # itself where that is not small against the mean's square.
    k = (64 + ch / 1024) * 2.0 ** -24
    xs, r = _up(x), wr.detach()[:, None]
    level = xs.abs().mean(1, keepdim=True)
    off = (xs - xs.mean(1, keepdim=True)).abs() + level
    # The relative error of rstd: half that of the variance.
    rel_r = 2 * k * (off.square().mean(1, keepdim=True) * r * r)
    hat = off * r * (1 + rel_r / k)
    R.check(mean, wm.detach(), level[:, 0], k, "mean")
    R.check(rstd, wr.detach(), (wr.detach() * (1 + rel_r[:, 0] / k)), k, "rstd")
    R.check(y, wy.detach(), hat * leaf[1].detach().abs() + leaf[2].detach().abs(), 2 * k, "y")
    d, aw = _up(dy).abs(), leaf[1].detach().abs()
    m0, m1 = (d * aw).mean(1, keepdim=True), (d * aw * hat).mean(1, keepdim=True)
    R.check(dx, gx, r * (1 + rel_r / k) * (d * aw + m0 + hat * m1), 6 * k, "dx")
    more = rows * 2.0 ** -24
    R.check(dw, gw, (d * hat).sum(0), 2 * k + more, "dw")
    R.check(db, gb, d.sum(0), k + more, "db")
    first = [t.clone() for t in (dx, dw, db)]
    cuda_device.layer_norm_backward_device(*args, weight=w, dweight=dw, dbias=db, stream=_stream())
    assert all(torch.equal(p, q) for p, q in zip(first, (dx, dw, db)))


def test_norm_without_parameters_and_statistics(cuda_device):
    g = _gen(3)
    x = _rows(g, 6, 96, torch.float32)
    y, z = torch.empty_like(x), torch.empty_like(x)
    cuda_device.layer_norm_device(x, y, stream=_stream())
    cuda_device.layer_norm_device(x, z, weight=torch.ones(96).cuda(), bias=torch.zeros(96).cuda(), stream=_stream())
    assert torch.equal(y, z)
    half = x.to(torch.bfloat16)
    w = torch.randn(96, generator=g).cuda()
    p, q = torch.empty_like(half), torch.empty_like(half)
    cuda_device.layer_norm_device(half, p, weight=w.to(torch.bfloat16), stream=_stream())
    cuda_device.layer_norm_device(half, q, weight=w.to(torch.bfloat16).float(), stream=_stream())
    assert torch.equal(p, q)


def test_norm_constant_and_non_finite_rows(cuda_device):
    x = torch.full((4, 64), 3.25, device="cuda")
    x[1, 5] = float("inf")
    x[2, 7] = NAN
    y, mean, rstd = torch.empty_like(x), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    cuda_device.layer_norm_device(x, y, eps=1e-5, mean=mean, rstd=rstd, stream=_stream())
    assert (y[0] == 0).all() and (y[3] == 0).all() and mean[0] == 3.25
    assert torch.isnan(y[1]).any() and torch.isnan(y[2]).all()


def test_norm_far_rows(cuda_device):
    """Rows whose offsets pass 2^31 values."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("the rows do not fit this GPU")
    wide = torch.empty(36000, 65536, dtype=torch.bfloat16, device="cuda")
    x = wide[:, 100 * 8:100 * 8 + 256]
    x.copy_(torch.randn(36000, 256, device="cuda"))
    y, z = torch.empty(36000, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(36000, 256, dtype=torch.bfloat16, device="cuda")
    cuda_device.layer_norm_device(x, y, stream=_stream())
    cuda_device.layer_norm_device(x.contiguous(), z, stream=_stream())
    assert torch.equal(y, z)


def test_norm_of_more_than_half_a_billion_rows(cuda_device):
    rows = (1 << 29) + 8
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("the rows do not fit this GPU")
    x = torch.randn(rows, 1, dtype=torch.bfloat16, device="cuda")
    y, mean = torch.ones_like(x), torch.zeros(rows, device="cuda")
    cuda_device.layer_norm_device(x, y, mean=mean, stream=_stream())
    assert (y == 0).all() and torch.equal(mean, x[:, 0].float())
    del x, y, mean
    torch.cuda.empty_cache()


# ---- streams, graphs, refusals, and the operators together ----------------------------------------------


def test_captured_and_replayed(cuda_device):
    """A captured pass replays on new inputs with the bits of the eager one; two graphs have workspaces of their own."""
    passes = []
    for seed in (11, 12):
        s = Scan([90, 0, 130, 40], 72, 16, dtype=torch.bfloat16, state=True, seed=seed)
        v = Conv(s.lens, 72, 4, torch.bfloat16, seed=seed)
        marks = s.marks(cuda_device)
        mid, out, final, dx = (torch.zeros_like(s.x) for _ in range(2)), {}, torch.zeros_like(s.state), torch.zeros_like(s.x)
        mid, y = mid
        scan_room = _room(cuda_device.selective_scan_workspace(s.tokens, 72, 16, 4, 1))
        back_room = _room(cuda_device.selective_scan_backward_workspace(s.tokens, 72, 16, 4, 1))
        ddt, da, db, dc, dz = (torch.zeros_like(s.x), torch.zeros_like(s.a), torch.zeros(s.b.shape, dtype=s.dtype, device="cuda"),
                               torch.zeros(s.b.shape, dtype=s.dtype, device="cuda"), torch.zeros_like(s.x))

        def run(s=s, v=v, marks=marks, mid=mid, y=y, final=final, scan_room=scan_room, back_room=back_room, dx=dx, ddt=ddt, da=da,
                db=db, dc=dc, dz=dz):
            st = torch.cuda.current_stream()
            cuda_device.causal_conv_device(v.x, v.w, mid, bias=v.bias, silu=True, seq_ptr=v.ptr, stream=st)
            cuda_device.selective_scan_device(mid, s.dt, s.a, s.b, s.c, y, scan_room, d=s.d, z=s.z, dt_bias=s.bias, softplus=True,
                                              seq_ptr=s.ptr, state=s.state, final_state=final, checkpoints=marks, stream=st)
            cuda_device.selective_scan_backward_device(s.dy, mid, s.dt, s.a, s.b, s.c, marks, dx, ddt, da, db, dc, back_room, d=s.d,
                                                       z=s.z, dz=dz, dt_bias=s.bias, softplus=True, seq_ptr=s.ptr, state=s.state,
                                                       dfinal_state=s.dfinal, stream=st)
            return y, final, dx, ddt, da, db, dc, dz

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        passes.append((s, v, run, graph, outs))
    for s, v, *_ in passes:
        v.x.copy_(torch.randn(v.x.shape, device="cuda"))
    for *_, graph, _ in passes:
        graph.replay()
    torch.cuda.synchronize()
    for s, v, run, graph, outs in passes:
        got = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_other_streams(cuda_device):
    """A stream of its own, a stream's handle, and the device's own stream give the same bits."""
    s = Scan([100, 60], 30, 16, dtype=torch.float16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y1 = s.forward(cuda_device, stream=side)
        y2 = s.forward(cuda_device, stream=side.cuda_stream)
    side.synchronize()
    y3 = torch.zeros_like(y1)
    room = _room(cuda_device.selective_scan_workspace(s.tokens, 30, 16, 2, 1))
    torch.cuda.synchronize()
    cuda_device.selective_scan_device(s.x, s.dt, s.a, s.b, s.c, y3, room, d=s.d, z=s.z, dt_bias=s.bias, softplus=True, seq_ptr=s.ptr)
    cuda_device.wait()
    assert torch.equal(y1, y2) and torch.equal(y1, y3)


def test_far_token_rows(cuda_device):
    """Convolution and scan, forward and gradients, over column ranges of arrays whose rows pass 2^32 bytes and 2^31 values
    give the bits that they give over contiguous rows."""
    dev, st = cuda_device, _stream()
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("the rows do not fit this GPU")
    t, ch, ns, dtype = 36000, 32, 8, torch.bfloat16
    g = _gen(6)
    lens = [9000, 1, 26900]  # 99 rows of no sequence
    ptr = torch.tensor(R.lengths_to_ptr(lens), dtype=torch.int32).cuda()
    wide = torch.zeros(t, 65536, dtype=dtype, device="cuda")
    far = [wide[:, 800 * 64 + k * 64:][:, :ch] for k in range(10)]  # x, dt, z, dy, y, dx, ddt, dz, v, dv
    near = [torch.zeros(t, ch, dtype=dtype, device="cuda") for _ in far]
    for k in range(4):
        near[k].copy_(torch.randn(t, ch, generator=g))
        far[k].copy_(near[k])
    b, c = torch.randn(t, ns, generator=g).to(dtype).cuda(), torch.randn(t, ns, generator=g).to(dtype).cuda()
    a, w = -torch.rand(ch, ns, generator=g).cuda() - 0.5, torch.randn(ch, 4, generator=g).cuda()
    marks = _room(dev.selective_scan_checkpoints(t, ch, ns))
    room = _room(max(dev.selective_scan_workspace(t, ch, ns, 3), dev.selective_scan_backward_workspace(t, ch, ns, 3),
                     dev.causal_conv_backward_workspace(t, ch, 4)))

    def run(x, dt, z, dy, y, dx, ddt, dz, v, dv):
        da, db, dc, dw = torch.empty_like(a), torch.zeros_like(b), torch.zeros_like(c), torch.empty_like(w)
        dev.causal_conv_device(x, w, v, silu=True, seq_ptr=ptr, stream=st)
        dev.selective_scan_device(v, dt, a, b, c, y, room, z=z, softplus=True, seq_ptr=ptr, checkpoints=marks, stream=st)
        dev.selective_scan_backward_device(dy, v, dt, a, b, c, marks, dv, ddt, da, db, dc, room, z=z, dz=dz, softplus=True,
                                           seq_ptr=ptr, stream=st)
        dev.causal_conv_backward_device(dv, x, w, dx, dw, room, silu=True, seq_ptr=ptr, stream=st)
        return da, db, dc, dw

    first, second = run(*near), run(*far)
    for p, q in zip((*near, *first), (*far, *second)):
        assert torch.equal(p, q) and torch.isfinite(p).all()
    assert far[4][30000:35000].abs().max() > 0 and (far[4][sum(lens):] == 0).all()
    del wide, far, p, q
    torch.cuda.empty_cache()


def test_replayed_with_other_sequences(cuda_device):
    """A captured prompt reads seq_ptr, slots and resume when it runs: replayed with others it gives what a call with them gives."""
    dev = cuda_device
    s, v = Scan([90, 0, 130, 40, 60], 72, 16, dtype=torch.bfloat16), Conv([90, 0, 130, 40, 60], 72, 4, torch.bfloat16)
    slots, resume = torch.tensor([3, 0, 5, 1, 6], dtype=torch.int32).cuda(), torch.tensor([1, 0, 1, 0, 1], dtype=torch.uint8).cuda()
    pool, cpool = torch.randn(8, 72, 16, device="cuda"), torch.randn(8, 3, 72, device="cuda").to(torch.bfloat16)
    keep = pool.clone(), cpool.clone()
    y, u = torch.zeros_like(s.x), torch.zeros_like(s.x)
    room = _room(dev.selective_scan_workspace(s.tokens, 72, 16, 5, 1))

    def run():
        st = torch.cuda.current_stream()
        dev.causal_conv_device(v.x, v.w, u, bias=v.bias, seq_ptr=s.ptr, state=cpool, final_state=cpool, slots=slots, resume=resume,
                               stream=st)
        dev.selective_scan_device(u, s.dt, s.a, s.b, s.c, y, room, d=s.d, z=s.z, dt_bias=s.bias, softplus=True, seq_ptr=s.ptr,
                                  state=pool, final_state=pool, slots=slots, resume=resume, stream=st)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for starts, rows, begin in (([0, 90, 90, 220, 260, 320], [3, 0, 5, 1, 6], [1, 0, 1, 0, 1]),
                                ([2, 3, 200, 200, 201, 310], [0, -1, 7, 2, 4], [0, 1, 1, 1, 0]),
                                ([0, 0, 0, 320, 320, 320], [1, 2, 3, 4, 5], [1, 1, 1, 1, 1])):
        s.ptr.copy_(torch.tensor(starts))
        slots.copy_(torch.tensor(rows))
        resume.copy_(torch.tensor(begin))
        got = []
        for go in (graph.replay, run):
            pool.copy_(keep[0])
            cpool.copy_(keep[1])
            y.fill_(7)
            u.fill_(7)
            go()
            torch.cuda.synchronize()
            got.append([t.clone() for t in (y, u, pool, cpool)])
        assert all(torch.equal(p, q) for p, q in zip(*got))
        assert (got[0][0][:starts[0]] == 7).all() and (got[0][0][starts[-1]:] == 7).all()


def test_the_default_streams_handle_is_that_stream(cuda_device):
    """A call on the handle of torch's default stream, 0, follows the work that makes its inputs there."""
    x, y = torch.zeros(4096, 4096, device="cuda"), torch.zeros(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for k in range(1, 4):
        for _ in range(40):  # some milliseconds of work in front of the input
            x.add_(1.0)
        x.copy_(torch.arange(4096, device="cuda", dtype=torch.float32).expand(4096, 4096) * k)
        cuda_device.layer_norm_device(x, y, eps=0.0, stream=torch.cuda.default_stream().cuda_stream)
        want = y.clone()
        torch.cuda.synchronize()
        cuda_device.layer_norm_device(x, y, eps=0.0)
        cuda_device.wait()
        assert torch.equal(want, y) and torch.isfinite(y).all()


def test_two_threads_at_once(cuda_device):
    """Calls from two threads, each on its own stream with its own arrays, give what they give alone."""
    import threading

    sets = [Scan([120, 33, 70], 64, 16, dtype=torch.bfloat16, state=True, seed=k) for k in (21, 22)]
    marks = [s.marks(cuda_device) for s in sets]
    alone = [(s.forward(cuda_device, marks=m, state=s.state), s.backward(cuda_device, m)) for s, m in zip(sets, marks)]
    torch.cuda.synchronize()
    failed = []

    def work(s, m, want):
        try:
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                for _ in range(10):
                    y = s.forward(cuda_device, marks=m, state=s.state, stream=side)
                    got = s.backward(cuda_device, m, stream=side)
            side.synchronize()
            assert torch.equal(y, want[0]) and all(torch.equal(v, want[1][k]) for k, v in got.items())
        except Exception as e:  # noqa: BLE001 (reported by the main thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(sets, marks, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_norms_of_two_widths_from_two_threads(cuda_device):
    """Widths that share a kernel but not its shared memory's size, called at once."""
    import threading

    sets = []
    for ch in (2056, 4096):
        x = torch.randn(2400, ch, device="cuda")
        y = torch.zeros_like(x)
        cuda_device.layer_norm_device(x, y, stream=_stream())
        sets.append((x, y))
    torch.cuda.synchronize()
    failed = []

    def work(x, want):
        try:
            side, y = torch.cuda.Stream(), torch.zeros_like(x)
            for _ in range(3000):
                cuda_device.layer_norm_device(x, y, stream=side)
            side.synchronize()
            assert torch.equal(y, want)
        except Exception as e:  # noqa: BLE001 (reported by the main thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=a) for a in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_current_device_is_kept(cuda_device):
    """A call leaves the thread's current device and its torch stream as they were, and nothing allocated."""
    s = Scan([64], 32, 16, ragged=False)
    y, room = torch.zeros_like(s.x), _room(cuda_device.selective_scan_workspace(64, 32, 16, 1, 1))
    torch.cuda.synchronize()
    before = (torch.cuda.current_device(), torch.cuda.mem_get_info()[0], torch.cuda.memory_allocated())
    for _ in range(3):
        cuda_device.selective_scan_device(s.x, s.dt, s.a, s.b, s.c, y, room, stream=_stream())
    torch.cuda.synchronize()
    assert before == (torch.cuda.current_device(), torch.cuda.mem_get_info()[0], torch.cuda.memory_allocated())


def test_sequence_starts_outside_the_tokens_are_clamped(cuda_device):
    """No content of seq_ptr or slots leads an access out of the arrays: their neighbours stay as they are."""
    s, v = Scan([40, 30, 26], 20, 16, state=True), Conv([40, 30, 26], 20, 4, state=True)
    for bad in ([0, 1000000, 2000000, 2147483647], [-7, -3, 50, 96], [90, 10, 60, 20], [96, 96, 96, 96], [0, 0, 0, 0]):
        ptr = torch.tensor(bad, dtype=torch.int32).cuda()
        s.ptr = v.ptr = ptr
        guard = torch.full((s.tokens + 4, 20), 5.0, device="cuda")
        y = guard[2:-2]
        pool = torch.cat([torch.full((1, 20, 16), 5.0, device="cuda"), s.state, torch.full((1, 20, 16), 5.0, device="cuda")])
        cpool = torch.cat([torch.full((1, 3, 20), 5.0, device="cuda"), v.state, torch.full((1, 3, 20), 5.0, device="cuda")])
        room = _room(cuda_device.selective_scan_workspace(s.tokens, 20, 16, 3, 1))
        cuda_device.selective_scan_device(s.x, s.dt, s.a, s.b, s.c, y, room, seq_ptr=ptr, softplus=True, state=pool[1:4],
                                          final_state=pool[1:4], stream=_stream())
        cuda_device.causal_conv_device(v.x, v.w, y, seq_ptr=ptr, state=cpool[1:4], final_state=cpool[1:4], stream=_stream())
        s.backward(cuda_device, s.marks(cuda_device))
        v.backward(cuda_device)
        torch.cuda.synchronize()
        for t in (guard[:2], guard[-2:], pool[:1], pool[4:], cpool[:1], cpool[4:]):
            assert (t == 5).all()


def test_conv_gradients_of_starts_that_do_not_ascend(cuda_device):
    """A sequence that begins and ends in front of what its tile has done reads no row behind its final state's gradient;
    the outputs' neighbours stay as they are."""
    for ptr in ([23, 22, 15, 18, 17, 2, 0, 30], [40, 30, 0, 17, 16, 16, 40], [16, 31, 20, 24, 16, 18, 32, 17]):
        n = len(ptr) - 1
        v = Conv([40] + [0] * (n - 1), 33, 4, state=True)
        v.ptr = torch.tensor(ptr, dtype=torch.int32).cuda()
        guard = torch.full((n + 2, 3, 33), 5.0, device="cuda")
        dx = torch.full((44, 33), 5.0, device="cuda")
        dw, room = torch.zeros_like(v.w), _room(cuda_device.causal_conv_backward_workspace(40, 33, 4))
        cuda_device.causal_conv_backward_device(v.dy, v.x, v.w, dx[2:-2], dw, room, bias=v.bias, silu=True, seq_ptr=v.ptr,
                                                state=v.state, dstate=guard[1:-1], dfinal_state=v.dfinal, stream=_stream())
        torch.cuda.synchronize()
        for t in (guard[:1], guard[-1:], dx[:2], dx[-2:]):
            assert (t == 5).all()
        assert torch.isfinite(dw).all()


def _refused(kind, call, *args, **kw):
    with pytest.raises(OpError) as e:
        call(*args, **kw)
    assert e.value.kind == kind, e.value
    return str(e.value)


def test_refusals(cuda_device):
    dev, st = cuda_device, _stream()
    s, v = Scan([40, 24], 20, 16, state=True), Conv([40, 24], 20, 4, state=True)
    y = torch.zeros_like(s.x)
    room = _room(dev.selective_scan_workspace(64, 20, 16, 2, 1))
    run = dev.selective_scan_device
    long = Scan([50, 46], 20, 16)
    assert "workspace" in _refused("Length", run, long.x, long.dt, long.a, long.b, long.c, torch.zeros_like(long.x), None,
                                   seq_ptr=long.ptr, stream=st)
    _refused("Backend", run, s.x, s.dt, s.a, s.b, s.c, s.x, room, stream=st)  # y over x
    _refused("Length", run, s.x, s.dt, s.a, s.b, s.c, y, room, n_seq=3, stream=st)  # 64 tokens in 3 equal parts
    _refused("Length", run, s.x, s.dt, s.a, s.b, s.c, y, room, seq_ptr=s.ptr, state=s.state[:1].clone(), stream=st)
    part = torch.zeros(3, 20, 16, device="cuda")
    _refused("Backend", run, s.x, s.dt, s.a, s.b, s.c, y, room, seq_ptr=s.ptr, state=part[:2], final_state=part[1:], stream=st)
    _refused("Backend", run, s.x.cpu(), s.dt, s.a, s.b, s.c, y, room, stream=st)  # host memory
    _refused("Length", run, s.x[:1].expand(64, 20), s.dt, s.a, s.b, s.c, y, room, stream=st)  # rows on top of one another
    _refused("Length", dev.selective_scan_device, s.x, s.dt, s.a, s.b, s.c, y, room, checkpoints=_room(64), stream=st)
    odd = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")[4:]
    _refused("Backend", run, long.x, long.dt, long.a, long.b, long.c, torch.zeros_like(long.x), odd, seq_ptr=long.ptr, stream=st)
    wide = torch.zeros(20, 65, device="cuda")
    _refused("Length", run, s.x, s.dt, wide, torch.zeros(64, 65, device="cuda"), torch.zeros(64, 65, device="cuda"), y, room, stream=st)
    conv = dev.causal_conv_device
    _refused("Length", conv, v.x, torch.zeros(20, 5, device="cuda"), y, stream=st)  # width
    _refused("Length", conv, v.x, torch.zeros(20, 1, device="cuda"), y, stream=st)
    _refused("Backend", conv, v.x, v.w, v.x, stream=st)
    both = torch.zeros(64, 40, device="cuda")
    conv(both[:, :20], v.w, both[:, 20:], stream=st)  # halves of one array do not overlap
    _refused("Backend", conv, both[:, :20], v.w, both[:, 10:30], stream=st)
    norm = dev.layer_norm_device
    _refused("Backend", norm, v.x, v.x, stream=st)
    _refused("Backend", norm, v.x, y, eps=-1.0, stream=st)
    _refused("Length", dev.layer_norm_backward_device, v.dy, v.x, torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda"), y,
             None, stream=st)
    torch.cuda.synchronize()


def test_only_the_final_state_may_be_the_state(cuda_device):
    """Outputs that are the state's own bytes in another role are refused, equal sizes or not."""
    dev, st = cuda_device, _stream()
    ch, width = 16, 4
    v = Conv([3, 3], ch, width)  # 6 tokens: as many values as two states
    state = torch.zeros(2, width - 1, ch, device="cuda")
    y = state.view(6, ch)
    assert "overlap" in _refused("Backend", dev.causal_conv_device, v.x, v.w, y, seq_ptr=v.ptr, state=state, stream=st)
    _refused("Backend", dev.causal_conv_device, v.x, v.w, y, seq_ptr=v.ptr, final_state=state, stream=st)
    _refused("Backend", dev.causal_conv_device, v.x, v.w, y, seq_ptr=v.ptr, state=state, final_state=state, stream=st)
    s = Scan([4, 4], ch, 4)  # 8 tokens: as many values as two states
    state = torch.zeros(2, ch, 4, device="cuda")
    args = (s.x, s.dt, s.a, s.b, s.c)
    _refused("Backend", dev.selective_scan_device, *args, state.view(8, ch), seq_ptr=s.ptr, state=state, stream=st)
    _refused("Backend", dev.selective_scan_step_device, s.x[:2], s.dt[:2], s.a, s.b[:2], s.c[:2], state.view(8, ch)[:2], state, stream=st)
    torch.cuda.synchronize()
    assert (state == 0).all()


def test_gradients_of_interleaved_runs(cuda_device):
    """db and dc may interleave group by group, as b and c may: [tokens, groups, 2, states]; runs that meet are refused."""
    dev = cuda_device
    for tail in (0, 5):  # rows that hold whole groups only, and some columns more
        s = Scan([40, 3], 24, 8, groups=3, dtype=torch.bfloat16)
        marks = s.marks(dev)
        s.forward(dev, marks=marks)
        want = s.backward(dev, marks)
        wide = torch.full((43, 3 * 2 * 8 + tail), 7.0, dtype=torch.bfloat16, device="cuda")
        runs = wide[:, :48].unflatten(1, (3, 2, 8))
        out = {k: torch.zeros_like(want[k]) for k in ("dx", "ddt", "dz", "da", "dd", "ddt_bias")}
        room = _room(dev.selective_scan_backward_workspace(43, 24, 8, 2, 3))

        def run(db, dc):
            dev.selective_scan_backward_device(s.dy, s.x, s.dt, s.a, s.b, s.c, marks, out["dx"], out["ddt"], out["da"], db, dc, room,
                                               d=s.d, dd=out["dd"], z=s.z, dz=out["dz"], dt_bias=s.bias, ddt_bias=out["ddt_bias"],
                                               softplus=True, seq_ptr=s.ptr, stream=_stream())

        run(runs[:, :, 0], runs[:, :, 1])
        assert torch.equal(runs[:, :, 0], want["db"]) and torch.equal(runs[:, :, 1], want["dc"])
        run(runs[:, :, 1], runs[:, :, 0])
        assert torch.equal(runs[:, :, 1], want["db"]) and torch.equal(runs[:, :, 0], want["dc"])
        assert (wide[:, 48:] == 7).all()
        meet = wide[:, 1:1 + 40].unflatten(1, (5, 8))[:, ::2] if tail else wide[:, :40].unflatten(1, (5, 8))[:, ::2]
        _refused("Backend", run, runs[:, :, 0], meet)
    one = torch.zeros(1, 48, dtype=torch.bfloat16, device="cuda").unflatten(1, (3, 2, 8))  # a single token
    s = Scan([1], 24, 8, groups=3, dtype=torch.bfloat16)
    marks = s.marks(dev)
    s.forward(dev, marks=marks)
    want = s.backward(dev, marks)
    dx, ddt, dz, da = (torch.zeros_like(v) for v in (s.x, s.x, s.x, s.a))
    room = _room(dev.selective_scan_backward_workspace(1, 24, 8, 1, 3))
    dev.selective_scan_backward_device(s.dy, s.x, s.dt, s.a, s.b, s.c, marks, dx, ddt, da, one[:, :, 0], one[:, :, 1], room, d=s.d, z=s.z,
                                       dz=dz, dt_bias=s.bias, softplus=True, seq_ptr=s.ptr, stream=_stream())
    assert torch.equal(one[:, :, 0], want["db"]) and torch.equal(one[:, :, 1], want["dc"])


def test_a_layer_of_them(cuda_device):
    """norm -> projection -> convolution -> projection -> scan, its gradients against autograd in 64 bits, and a token more
    through the kept states against the prompt that holds it."""
    dev, st = cuda_device, _stream()
    g = _gen(42)
    lens, width, ch, ns, rank = [37, 60, 1, 30], 24, 48, 8, 6
    t = sum(lens)
    ptr = torch.tensor(R.lengths_to_ptr(lens), dtype=torch.int32).cuda()
    put = lambda *shape, k=1.0: (torch.randn(*shape, generator=g) * k).cuda()  # noqa: E731
    u, dy = put(t, width), put(t, ch)
    nw, nb = 1 + put(width, k=0.1), put(width, k=0.1)
    w_in, w_x, w_dt = put(2 * ch, width, k=width ** -0.5), put(rank + 2 * ns, ch, k=ch ** -0.5), put(ch, rank, k=rank ** -0.5)
    cw, cb = put(ch, 4, k=0.5), put(ch, k=0.1)
    a = -torch.exp(put(ch, ns, k=0.3))
    d, bias = put(ch), put(ch, k=0.5) - 2

    def forward(u, ptr, seqs, conv_state=None, scan_state=None):
        rows = u.shape[0]
        n, mean, rstd = torch.empty_like(u), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        dev.layer_norm_device(u, n, weight=nw, bias=nb, mean=mean, rstd=rstd, stream=st)
        xz = n @ w_in.t()
        x, z, v, y = xz[:, :ch], xz[:, ch:], torch.empty(rows, ch, device="cuda"), torch.empty(rows, ch, device="cuda")
        dev.causal_conv_device(x, cw, v, bias=cb, silu=True, seq_ptr=ptr, final_state=conv_state, stream=st)
        p = v @ w_x.t()
        dt = p[:, :rank] @ w_dt.t()
        b, c = p[:, rank:rank + ns], p[:, rank + ns:]
        marks = _room(dev.selective_scan_checkpoints(rows, ch, ns))
        room = _room(max(dev.selective_scan_workspace(rows, ch, ns, seqs), dev.selective_scan_backward_workspace(rows, ch, ns, seqs)))
        dev.selective_scan_device(v, dt, a, b, c, y, room, d=d, z=z, dt_bias=bias, softplus=True, seq_ptr=ptr, final_state=scan_state,
                                  checkpoints=marks, stream=st)
        return y, (n, mean, rstd, x, z, v, p, dt, b, c, marks, room)

    y, (n, mean, rstd, x, z, v, p, dt, b, c, marks, room) = forward(u, ptr, 4)
    dxz, dp, dv, ddt = torch.empty(t, 2 * ch, device="cuda"), torch.empty_like(p), torch.empty_like(v), torch.empty_like(v)
    da, dd, dbias = torch.empty_like(a), torch.empty_like(d), torch.empty_like(bias)
    dev.selective_scan_backward_device(dy, v, dt, a, b, c, marks, dv, ddt, da, dp[:, rank:rank + ns], dp[:, rank + ns:], room, d=d,
                                       dd=dd, z=z, dz=dxz[:, ch:], dt_bias=bias, ddt_bias=dbias, softplus=True, seq_ptr=ptr, stream=st)
    dp[:, :rank] = ddt @ w_dt
    dv += dp @ w_x
    dcw, dcb = torch.empty_like(cw), torch.empty_like(cb)
    croom = _room(dev.causal_conv_backward_workspace(t, ch, 4))
    dev.causal_conv_backward_device(dv, x, cw, dxz[:, :ch], dcw, croom, bias=cb, dbias=dcb, silu=True, seq_ptr=ptr, stream=st)
    dn = dxz @ w_in
    du, dnw, dnb = torch.empty_like(u), torch.empty_like(nw), torch.empty_like(nb)
    dev.layer_norm_backward_device(dn, u, mean, rstd, du, _room(dev.layer_norm_backward_workspace(t, width)), weight=nw, dweight=dnw,
                                   dbias=dnb, stream=st)
    leaf = [_up(k).requires_grad_() for k in (u, nw, nb, cw, cb, a, d, bias)]
    ou, onw, onb, ocw, ocb, oa, od, obias = leaf
    on = R.norm(ou, onw, onb, 1e-5)[0]
    oxz = on @ _up(w_in).t()
    ov = R.conv(oxz[:, :ch], ocw, ocb, True, lens, None)[0]
    op = ov @ _up(w_x).t()
    odt = op[:, :rank] @ _up(w_dt).t()
    oy = R.scan(ov, odt, oa, op[:, None, rank:rank + ns], op[:, None, rank + ns:], od, oxz[:, ch:], obias, True, lens, None)[0]
    want = torch.autograd.grad((oy * _up(dy)).sum(), leaf)
    # Norm-wise: each stage rounds at 2^-24 (2^-22 an exponential) along at most 60 tokens each way, and the projections'
    # products may be computed in tf32 only where the program asks for it; 2^-14 leaves a factor of ten over 2 * 60 * 2^-22.
    near = lambda p, q: float((p.detach().cpu().to(F64) - q).norm() / q.norm())  # noqa: E731
    assert near(y, oy.detach()) < 2.0 ** -14
    for got, exp in zip((du, dnw, dnb, dcw, dcb, da, dd, dbias), want):
        assert near(got, exp) < 2.0 ** -14
    # The first sequence's tokens but the last as a prompt, then the last as a step.
    short = torch.tensor([0, lens[0] - 1], dtype=torch.int32).cuda()
    cst, sst = torch.empty(1, 3, ch, device="cuda"), torch.empty(1, ch, ns, device="cuda")
    forward(u[:lens[0] - 1], short, 1, cst, sst)
    one = u[lens[0] - 1:lens[0]]
    n1, v1, y1 = torch.empty_like(one), torch.empty(1, ch, device="cuda"), torch.empty(1, ch, device="cuda")
    dev.layer_norm_device(one, n1, weight=nw, bias=nb, stream=st)
    xz1 = n1 @ w_in.t()
    dev.causal_conv_step_device(xz1[:, :ch], cw, v1, cst, bias=cb, silu=True, stream=st)
    p1 = v1 @ w_x.t()
    dev.selective_scan_step_device(v1, p1[:, :rank] @ w_dt.t(), a, p1[:, rank:rank + ns], p1[:, rank + ns:], y1, sst, d=d,
                                   z=xz1[:, ch:], dt_bias=bias, softplus=True, stream=st)
    assert near(y1, oy.detach()[lens[0] - 1:lens[0]]) < 2.0 ** -14


def test_gradients_against_differences(cuda_device):
    """Along a random direction of all inputs, the scan's gradients give the change of its result in 64 bits."""
    s = Scan([21, 40], 12, 16, state=True, seed=9)
    marks = s.marks(cuda_device)
    s.forward(cuda_device, marks=marks, state=s.state)
    got = s.backward(cuda_device, marks)
    g = _gen(77)
    leaf = {"x": s.x, "dt": s.dt, "a": s.a, "b": s.b, "c": s.c, "d": s.d, "z": s.z, "dt_bias": s.bias, "start": s.state}
    names = {"x": "dx", "dt": "ddt", "a": "da", "b": "db", "c": "dc", "d": "dd", "z": "dz", "dt_bias": "ddt_bias", "start": "dstate"}
    dirs = {k: torch.randn(v.shape, generator=g, dtype=F64) for k, v in leaf.items()}

    def loss(eps):
        y, final = R.scan(softplus=True, lens=s.lens, **{k: _up(v) + eps * dirs[k] for k, v in leaf.items()})
        return float((y * _up(s.dy)).sum() + (final * _up(s.dfinal)).sum())

    slope = sum(float((_up(got[names[k]]) * dirs[k]).sum()) for k in leaf)
    size = sum(float((_up(got[names[k]]) * dirs[k]).abs().sum()) for k in leaf)
    h = 1e-5  # the differences' own error is of the order of h^2 and of 2^-52 / h
    diff = (loss(h) - loss(-h)) / (2 * h)
    _, k = s.oracle(s.state, backward=True)
    assert abs(slope - diff) <= (k + 1e-6) * size
