"""adamw_step and the optimizer AdamW against the formulas in 64 bits, with moments in 32 and in 8 bits; refusals, state
dicts, use by the Trainer.

Tolerances, u = 2^-24 (one fp32 rounding).  m' = m + c1 (g - m): the difference, the constant and the sum round:
u (|m'| + 2 c1 |g - m|).  v': b2 and its product, three factors of c2 g^2, the sum: u (2 b2 v + 3 c2 g^2 + v').
p': the constant 1 - lr wd, its product and the sum: u (2 |p| + |p'|); the update D = s m' / (sqrt(v') / sqrt(bc2) + eps): the
error of m' times s / denominator, and 20 u |D| for half of v's, the 1-ulp square root and reciprocal and five roundings.
A bf16 parameter adds half a step of its type.  An 8-bit moment may differ from the oracle's only where the random bits
decide within 2^-16 of a step (the value is off by at most 8 u, a step is at least 1/16 of it)."""
import copy
import math

import pytest
import torch

U = 2.0**-24
B1, B2, EPS, WD, LR = 0.9, 0.999, 1e-8, 0.01, 2e-3


def mix(x):
    x = ((x ^ (x >> 16)) * 0x21F0AAAD) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x735A2D97) & 0xFFFFFFFF
    return x ^ (x >> 15)


def chances(seed, tensor, step, index):
    """The two 16-bit numbers of each element, as fractions."""
    key = mix((mix((seed + 0x9E3779B9 * (tensor + 1)) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    seg = index >> 32
    keys = torch.where(seg > 0, mix((key + seg * 0x9E3779B9) & 0xFFFFFFFF), key)
    h = mix((index & 0xFFFFFFFF) ^ keys)
    return (h & 0xFFFF).double() / 65536, (h >> 16).double() / 65536


def decode(codes, scales):
    s = scales.view(torch.uint8).double()
    value = codes.view(torch.float8_e4m3fn).flatten().float().double()
    return value * torch.exp2(s - 127).repeat_interleave(128)[: value.numel()]


def scale_ref(x):
    """Biased exponent per 128 elements: the least E >= -126 with max <= 448 * 2^E; finite values count."""
    n = x.numel()
    b = torch.nn.functional.pad(torch.where(torch.isfinite(x), x.abs(), 0.0), (0, -n % 128)).view(-1, 128).amax(-1)
    e = torch.ceil(torch.log2(b.clamp(min=1e-300) / 448)).clamp(-126, 127)
    return torch.where(b > 0, e + 127, 0.0)


def check_8bit(codes, scales, x, u, keep):
    """codes / scales against the value x (64 bits) rounded with the chances u."""
    s = scale_ref(x)
    got_s = scales.view(torch.uint8).double()
    assert torch.equal(got_s, s), (got_s - s).abs().max()
    n = x.numel()
    unit = torch.exp2(s - 127).repeat_interleave(128)[:n]
    empty = (s == 0).repeat_interleave(128)[:n]
    y = torch.where(empty, 0.0, x / unit).abs()
    step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0**-6))) - 3)
    place = y / step + u
    want = torch.floor(place) * step
    if keep:
        want = torch.where((want == 0) & (y > 0), 2.0**-9, want)
    got = codes.view(torch.float8_e4m3fn).flatten().float().double()
    fin = torch.isfinite(x)
    assert torch.equal(torch.isnan(got), ~fin)
    differ = fin & (got.abs() != want)
    near = (place - torch.round(place)).abs() < 2.0**-16
    assert not (differ & ~near).any(), int((differ & ~near).sum())
    assert int(differ.sum()) <= 2 + n // 1000
    assert ((got.sign() == x.sign()) | (got == 0) | ~fin).all()


def make(shape, pdt, gdt, eight, seed, lead=0):
    """A parameter, a gradient (some rows zero) and moments; lead: elements before the view's first."""
    g = torch.Generator().manual_seed(seed)
    n = math.prod(shape)
    size = torch.exp(2 * torch.randn(n // 64 + 1, generator=g)).repeat_interleave(64)[:n]
    size = size * (torch.rand(n // 64 + 1, generator=g) > 0.2).repeat_interleave(64)[:n]

    def on_gpu(t, dtype):
        big = torch.zeros(n + lead, dtype=dtype, device="cuda")
        big[lead:] = t.to("cuda", dtype)
        return big[lead:].view(shape)

    p, gr = on_gpu(0.1 * torch.randn(n, generator=g), pdt), on_gpu(1e-3 * size * torch.randn(n, generator=g), gdt)
    m, r = 3e-4 * size * torch.randn(n, generator=g), 1e-3 * size * (0.1 + torch.rand(n, generator=g))
    if not eight:
        return p, gr, on_gpu(m, torch.float32), on_gpu(r * r, torch.float32)
    out = []
    for x in (m, r):
        s = scale_ref(x.double())
        y = x / torch.exp2(s - 127).repeat_interleave(128)[:n].float()
        c = on_gpu(torch.where((s == 0).repeat_interleave(128)[:n], 0.0, y).to(torch.float8_e4m3fn).view(torch.uint8), torch.uint8)
        out.append((c, s.to(torch.uint8).cuda()))
    return p, gr, out[0], out[1]


def oracle_and_check(before, after, pos, step, seed, lr=LR, wd=WD, b1=B1, b2=B2, eps=EPS):
    """before: (p, g, m, v) copies; after: (p, m, v) as the call left them."""
    p, g, m, v = before
    p2, m2, v2 = after
    eight = isinstance(m, tuple)
    p, g = p.double().flatten(), g.double().flatten()
    m = decode(*m) if eight else m.double().flatten()
    v = decode(*v) ** 2 if eight else v.double().flatten()
    m_new, v_new = m + (1 - b1) * (g - m), b2 * v + (1 - b2) * g * g
    # v is an fp32 value: what lies below half of fp32's least number, 2^-150, is 0 whichever way the product is formed (each of
    # its roundings moves a value of this size by at most 2^-150, and here the terms are 2^-156 and less, or none)
    assert not ((v_new > 2.0**-156) & (v_new < 2.0**-120)).any()
    v_new = torch.where(v_new < 2.0**-150, 0.0, v_new)
    s = lr / (1 - b1**step)
    den = torch.sqrt(v_new) / math.sqrt(1 - b2**step) + eps
    D = s * m_new / den
    p_new = p * (1 - lr * wd) - D
    m_room = U * (m_new.abs() + 2 * (1 - b1) * (g - m).abs())
    p_room = U * (2 * p.abs() + p_new.abs() + 20 * D.abs()) + s * m_room / den
    if p2.dtype == torch.bfloat16:
        p_room = p_room + torch.finfo(torch.bfloat16).eps / 2 * (p_new.abs() + p_room)
    fin = torch.isfinite(p_new)
    got = p2.double().flatten()
    assert torch.equal(torch.isfinite(got), fin)
    assert ((got - p_new).abs() <= p_room)[fin].all(), ((got - p_new).abs() / p_room)[fin].max()
    if eight:
        lo, hi = chances(seed, pos, step, torch.arange(p.numel(), device=p.device))
        check_8bit(*m2, m_new, lo, False)
        check_8bit(*v2, torch.sqrt(v_new), hi, True)
    else:
        assert ((m2.double().flatten() - m_new).abs() <= m_room + 1e-45)[fin].all()
        v_room = U * (2 * b2 * v + 3 * (1 - b2) * g * g + v_new) + 1e-44
        assert ((v2.double().flatten() - v_new).abs() <= v_room)[fin].all()


def copy_of(x):
    return tuple(t.clone() for t in x) if isinstance(x, tuple) else x.clone()


def run_and_check(tensors, step=7, seed=5, **kw):
    from clt_training_amd import hip_ops as ops

    before = [tuple(copy_of(t) for t in x) for x in tensors]
    ps, gs, ms, vs = (list(c) for c in zip(*tensors))
    ops.adamw_step(ps, gs, ms, vs, step=step, lr=kw.get("lr", LR), betas=(kw.get("b1", B1), kw.get("b2", B2)), eps=kw.get("eps", EPS),
                   weight_decay=kw.get("wd", WD), seed=seed)
    torch.cuda.synchronize()
    for i, (b, x) in enumerate(zip(before, tensors)):
        oracle_and_check(b, (x[0], x[2], x[3]), i, step, seed, **kw)


# ---------------------------------------------------------------------------------------------------------------- CPU
def test_refusals_without_a_gpu():
    from clt_training_amd import _lib, hip_ops as ops
    from clt_training_amd.adam import AdamW

    t = torch.zeros(4)
    with pytest.raises(ValueError, match="for every parameter"):
        ops.adamw_step([t], [], [t], [t], step=1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.adamw_step([t], [t], [t], [t], step=1)
    ops.adamw_step([], [], [], [], step=1)
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(t.clone())], **bad)
    lib = _lib.load()
    rec = (_lib.AdamWTensor * 1)()
    r = rec[0]
    r.p = r.g = r.m = r.v = 4096
    r.numel, r.lr = 8, 1e-3
    import ctypes as C

    call = lambda n=1, b1=0.9, b2=0.99, eps=1e-8, step=1: lib.clt_adamw_step(C.cast(rec, C.c_void_p), n, b1, b2, eps, step, 0, None)  # noqa: E731
    assert call(step=0) == -1 and b"counted from 1" in lib.clt_last_error()
    assert call(b1=1.0) == -1 and call(b2=-0.1) == -1 and call(n=-1) == -1
    assert lib.clt_adamw_step(None, 1, 0.9, 0.99, 1e-8, 1, 0, None) == -1
    r.m_scale = 4096
    assert call() == -1 and b"8 bits" in lib.clt_last_error()
    r.m_scale, r.m = None, 4098
    assert call() == -1 and b"misaligned" in lib.clt_last_error()
    r.m, r.p_dtype = 4096, 5
    assert call() == -1
    r.p_dtype, r.v = 0, None
    assert call() == -1
    r.v, r.numel = 4096, -1
    assert call() == -1


def test_c_refusal_of_a_tensor_too_large_for_a_launch():
    import ctypes as C

    from clt_training_amd import _lib

    rec = (_lib.AdamWTensor * 1)()
    rec[0].p = rec[0].g = rec[0].m = rec[0].v = 4096
    rec[0].numel = 2**35
    assert _lib.load().clt_adamw_step(C.cast(rec, C.c_void_p), 1, 0.9, 0.99, 1e-8, 1, 0, None) == -2


def test_trainer_takes_the_names_and_tp_refuses_them():
    from clt_training_amd import SparseCoderConfig, TrainConfig, Trainer
    from clt_training_amd.adam import AdamW
    from clt_training_amd.tp import TPTrainer

    for name, bits in (("adamw", 32), ("adamw8", 8)):
        cfg = TrainConfig(sae=SparseCoderConfig(k=4, expansion_factor=2, transcode=True), hookpoints=["a"], optimizer=name, weight_decay=0.1)
        opt = Trainer(cfg, [None] * 10, device="cpu", input_widths={"a": 8}).optimizers[0]
        assert type(opt) is AdamW and opt.state_bits == bits and opt.param_groups[0]["weight_decay"] == 0.1
        with pytest.raises(NotImplementedError, match="AdamW"):
            TPTrainer(cfg, [None] * 10, device="cpu", input_widths={"a": 8})
    cfg = TrainConfig(sae=SparseCoderConfig(k=4, expansion_factor=2, transcode=True, use_mxfp4=True), hookpoints=["a"], optimizer="adam")
    with pytest.raises(NotImplementedError, match="use_mxfp4"):
        TPTrainer(cfg, [None] * 10, device="cpu", input_widths={"a": 8})


def test_load_state_dict_keeps_types_and_refuses_what_does_not_fit():
    from clt_training_amd.adam import AdamW

    p = torch.nn.Parameter(torch.zeros(64, 128, dtype=torch.bfloat16))
    q = torch.nn.Parameter(torch.zeros(5))
    for bits in (8, 32):
        opt = AdamW([p, q], state_bits=bits)
        for t in (p, q):
            opt._moments(t)
        opt._step = 9
        new = AdamW([p, q], state_bits=bits)
        new.load_state_dict(opt.state_dict())
        assert new._step == 9 and {k: v.dtype for k, v in new.state[p].items()} == {k: v.dtype for k, v in opt.state[p].items()}
        assert all(a.data_ptr() != b.data_ptr() for a, b in zip(new.state[p].values(), opt.state[p].values()))
        other = AdamW([torch.nn.Parameter(torch.zeros(64, 127)), q], state_bits=bits)
        with pytest.raises(ValueError, match="does not fit"):
            other.load_state_dict(opt.state_dict())


def test_load_state_dict_of_torch():
    from clt_training_amd.adam import AdamW

    ps = [torch.nn.Parameter(torch.zeros(4, 5)), torch.nn.Parameter(torch.zeros(3))]
    ref = torch.optim.AdamW(ps, lr=0.1, weight_decay=0.2)
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn_like(p)
        ref.step()
    opt = AdamW(ps)
    opt.load_state_dict(ref.state_dict())
    assert opt._step == 3 and opt.param_groups[0]["weight_decay"] == 0.2
    assert all(torch.equal(opt.state[p]["exp_avg_sq"], ref.state[p]["exp_avg_sq"]) for p in ps)
    ref.state[ps[0]]["step"] += 1
    with pytest.raises(ValueError, match="one step count"):
        opt.load_state_dict(ref.state_dict())
    assert opt._step == 3
    with pytest.raises(ValueError, match="maximize"):
        opt.load_state_dict(torch.optim.AdamW(ps, maximize=True).state_dict())


def recorded(monkeypatch):
    """The calls that the optimizer makes, as {position in ``params``: step} each; nothing is computed."""
    from clt_training_amd import adam

    calls = []
    monkeypatch.setattr(adam, "adamw_step", lambda ps, *_, step, **kw: calls.append((list(ps), step)))
    return calls


def test_every_parameter_counts_its_own_steps(monkeypatch):
    """A parameter whose first gradient comes late starts at 1; steps without a gradient and refused calls count for nothing;
    the counts go through a state dict, also through the checkpoint's layout."""
    from clt_training_amd import adam, ckpt

    calls = recorded(monkeypatch)
    ps = [torch.nn.Parameter(torch.zeros(3)) for _ in range(3)]
    opt = adam.AdamW(ps[:2])
    opt.add_param_group(dict(params=ps[2:]))
    opt.step()
    assert not calls and opt._step == 0
    counts = [0, 0, 0]
    for grads in ([0], [0], [0, 2], [], [0, 1, 2], [1], [0, 1, 2]):
        for i, p in enumerate(ps):
            p.grad = torch.ones(3) if i in grads else None
        calls.clear()
        opt.step()
        seen = {next(i for i, p in enumerate(ps) if p is q): step for call, step in calls for q in call}
        for i in grads:
            counts[i] += 1
        assert seen == {i: counts[i] for i in grads}
    assert counts == [5, 3, 3] and opt._step == 6
    assert [len(c) for c, _ in calls] == [1, 2]  # (equal counts share a call, whatever group they are in)

    def fail(*_, **kw):
        raise ValueError("refused")

    monkeypatch.setattr(adam, "adamw_step", fail)
    with pytest.raises(ValueError, match="refused"):
        opt.step()
    assert opt._step == 6
    sd = opt.state_dict()
    assert [int(sd["state"][i]["step"]) for i in range(3)] == [5, 3, 3]
    nested, step = ckpt.from_file_layout(ckpt.to_reference_layout(sd, opt._step))
    for state in (sd, {**nested, "clt_step": step}):
        new = adam.AdamW(ps[:2])
        new.add_param_group(dict(params=ps[2:]))
        new.load_state_dict(state)
        calls = recorded(monkeypatch)
        new.step()
        assert {step: len(c) for c, step in calls} == {6: 1, 4: 2} and new._step == 7
        del new.state[ps[0]]  # (a parameter that begins anew)
        new.step()
        assert {step: len(c) for c, step in calls[2:]} == {1: 1, 5: 2}
    old = {**sd, "state": {i: {k: v for k, v in st.items() if k != "step"} for i, st in sd["state"].items()}}
    new.load_state_dict(old)  # (what was saved with one count for all)
    calls = recorded(monkeypatch)
    new.step()
    assert [(len(c), step) for c, step in calls] == [(3, 7)]


def test_counts_of_torch_are_taken_over(monkeypatch):
    """Equal counts as they are; counts that differ where the state says that they may."""
    from clt_training_amd import adam

    ps = [torch.nn.Parameter(torch.zeros(2)) for _ in range(2)]
    ref = torch.optim.AdamW(ps)
    for late in (None, None, torch.ones(2)):
        ps[0].grad, ps[1].grad = torch.ones(2), late
        ref.step()
    opt = adam.AdamW(ps)
    with pytest.raises(ValueError, match="clt_step"):
        opt.load_state_dict(ref.state_dict())
    opt.load_state_dict({**ref.state_dict(), "clt_step": 3})
    calls = recorded(monkeypatch)
    opt.step()
    assert [(c[0] is ps[0], len(c), step) for c, step in calls] == [(True, 1, 4), (False, 1, 2)]
    back = torch.optim.AdamW(ps)
    back.load_state_dict(opt.state_dict())
    assert [int(back.state[p]["step"]) for p in ps] == [4, 2]


def test_saved_weight_decay_is_decoupled_for_torch():
    """torch.optim.Adam goes on from a saved state, also from a checkpoint's file, as torch.optim.AdamW does; a state that an
    earlier version saved with the other label is put right when it is loaded."""
    from clt_training_amd import ckpt
    from clt_training_amd.adam import AdamW

    def ends(make, state):
        p = torch.nn.Parameter(torch.linspace(1, 2, 6))
        p.grad = torch.full((6,), 0.1)
        opt = make([p])
        opt.load_state_dict(copy.deepcopy(state))  # (torch steps on the tensors that it is given)
        opt.step()
        return p.detach()

    q = torch.nn.Parameter(torch.zeros(6))
    opt = AdamW([q], lr=1e-2, weight_decay=0.5)
    m, v = opt._moments(q)
    m.fill_(0.01), v.fill_(0.02)
    opt._steps[q], opt._step = 4, 4
    saved, step = ckpt.from_file_layout(ckpt.to_reference_layout(opt.state_dict(), opt._step))
    for state in (saved, opt.state_dict()):
        assert torch.equal(ends(torch.optim.Adam, state), ends(torch.optim.AdamW, state))
    for g in saved["param_groups"]:
        g["decoupled_weight_decay"] = False
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["decoupled_weight_decay"] is True and step == 4


def test_copies_go_on_where_the_optimizer_stands(monkeypatch):
    import pickle

    from clt_training_amd import adam

    ps = [torch.nn.Parameter(torch.zeros(n)) for n in (5000, 3)]
    opt = adam.AdamW(ps, lr=0.1, state_bits=8, seed=6)
    recorded(monkeypatch)
    for grads in ((1, 0), (1, 1)):
        for p, on in zip(ps, grads):
            p.grad = torch.ones_like(p) if on else None
        opt.step()
    opt.state[ps[0]]["rms_codes"].fill_(3)
    for new in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        qs = [q for g in new.param_groups for q in g["params"]]
        assert not any(p is q for p, q in zip(ps, qs)) and bool((new.state[qs[0]]["rms_codes"] == 3).all())
        for q in qs:
            q.grad = torch.ones_like(q)
        calls = []
        monkeypatch.setattr(adam, "adamw_step", lambda c, g, m, v, *, step, lr, seed, **kw: calls.append((len(c), type(m[0]) is tuple, step, lr[0], seed)))
        new.step()
        assert sorted(calls) == [(1, False, 2, 0.1, 6), (1, True, 3, 0.1, 6)] and new._step == 3 and opt._step == 2


def test_trainer_resumes_every_parameters_count(tmp_path):
    """Counts that differ go through a trainer's checkpoint."""
    from clt_training_amd import SparseCoderConfig, TrainConfig, Trainer

    def trainer():
        cfg = TrainConfig(sae=SparseCoderConfig(k=4, expansion_factor=2, transcode=True), hookpoints=["a"], optimizer="adamw")
        return Trainer(cfg, [None] * 10, device="cpu", input_widths={"a": 8})

    first = trainer()
    opt = first.optimizers[0]
    params = [p for g in opt.param_groups for p in g["params"]]
    for i, p in enumerate(params[:-1]):  # (the last one never had a gradient)
        opt._moments(p)
        opt._steps[p] = 3 + i % 2
    opt._step = 4
    first.save(tmp_path)
    again = trainer().load_state(tmp_path).optimizers[0]
    assert again._step == 4
    assert [again._steps.get(p) for g in again.param_groups for p in g["params"]] == [3 + i % 2 for i in range(len(params) - 1)] + [None]


# ---------------------------------------------------------------------------------------------------------------- GPU
SIZES = [(1,), (7,), (8,), (127,), (128,), (129,), (16, 8), (8191,), (8192,), (8193,), (33, 65), (257, 769)]


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("pdt,gdt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_step_against_64_bits(pdt, gdt, eight):
    run_and_check([make(s, pdt, gdt, eight, 10 + i) for i, s in enumerate(SIZES)])


@pytest.mark.gpu
def test_mixed_list_of_many_tensors():
    """More than one launch's worth, both kinds of moments, empty tensors, rates of their own, the first and a late step."""
    from clt_training_amd import hip_ops as ops

    for step in (1, 100000):
        ts = [make(((i * 37) % 300 + 1,), (torch.float32, torch.bfloat16)[i % 2], (torch.bfloat16, torch.float32)[i % 3 == 0], i % 5 == 0, i) for i in range(97)]
        ts[3] = tuple(torch.zeros(0, device="cuda") for _ in range(4))
        before = [tuple(copy_of(t) for t in x) for x in ts]
        lrs, wds = [1e-3 * (i + 1) for i in range(97)], [0.01 * (i % 3) for i in range(97)]
        ops.adamw_step(*(list(c) for c in zip(*ts)), step=step, lr=lrs, weight_decay=wds, seed=1)
        for i, (b, x) in enumerate(zip(before, ts)):
            if i != 3:
                oracle_and_check(b, (x[0], x[2], x[3]), i, step, 1, lr=lrs[i], wd=wds[i])


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_unaligned_views_and_neighbours(eight):
    """Views that start at any element; nothing before or behind them is written."""
    for lead in (1, 3, 8):
        for n in (5, 200, 9001):
            ts = [make((n,), pdt, gdt, eight, n + lead, lead) for pdt, gdt in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32))]
            run_and_check(ts)
            for t in ts:
                for x in (t[0], *((t[2][0], t[3][0]) if eight else (t[2], t[3]))):
                    whole = x.as_strided((lead,), (1,), 0)
                    assert (whole.float() == 0).all()
    # scales: the byte behind the last block
    from clt_training_amd import hip_ops as ops

    p, g, (mc, ms), (vc, vs) = make((130,), torch.float32, torch.float32, True, 1)
    guard = torch.full((2, 8), 77, dtype=torch.uint8, device="cuda")
    guard[0, :2], guard[1, :2] = ms, vs
    ops.adamw_step([p], [g], [(mc, guard[0, :2])], [(vc, guard[1, :2])], step=3)
    assert (guard[:, 2:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_zero_and_non_finite_gradients(eight):
    """Zero gradients on zero moments move nothing but the decay; NaN and infinity stay with their own element."""
    from clt_training_amd import hip_ops as ops

    p = torch.randn(1000, device="cuda")
    ref = p.clone()
    zero = lambda: tuple(torch.zeros(s, dtype=torch.uint8, device="cuda") for s in (1000, 8)) if eight else torch.zeros(1000, device="cuda")  # noqa: E731
    m, v, g = zero(), zero(), torch.zeros(1000, device="cuda")
    ops.adamw_step([p], [g], [m], [v], step=1, lr=0.1, weight_decay=0.5)
    assert torch.equal(p, ref * (1 - 0.05))
    for t in (*m, *v) if eight else (m, v):
        assert (t == 0).all()
    ts = make((1000,), torch.float32, torch.float32, eight, 3)
    ts[1][100], ts[1][300], ts[1][301] = float("nan"), float("inf"), 0.0
    run_and_check([ts])
    assert int((~torch.isfinite(ts[0])).sum()) == 2
    ts[1].zero_()  # the poison stays where it is
    run_and_check([ts], step=8)
    assert int((~torch.isfinite(ts[0])).sum()) == 2


@pytest.mark.gpu
def test_tiny_and_huge_moments():
    """Blocks at the ends of the scale's range, and values far below their block's maximum: r > 0 stays > 0."""
    g = torch.zeros(512, device="cuda")
    g[:128] = 1e-22 * torch.rand(128, device="cuda")
    g[128:256] = 1e17 * torch.rand(128, device="cuda")
    g[256], g[257:384] = 1.0, 1e-8
    m, v = ((torch.zeros(512, dtype=torch.uint8, device="cuda"), torch.zeros(4, dtype=torch.uint8, device="cuda")) for _ in range(2))
    p = torch.zeros(512, device="cuda")
    run_and_check([(p, g, m, v)], step=1, wd=0.0)
    r = decode(*v)
    assert (r[257:384] > 0).all() and (r[384:] == 0).all() and torch.isfinite(p).all()


@pytest.mark.gpu
def test_rounding_is_unbiased_and_lets_moments_decay():
    """600 steps without a gradient: r follows b2^(t/2).  A step rounds with a deviation of at most 1/8 r sqrt(q (1 - q)), q =
    0.0005 * 16 the share of a step that is lost: 0.011 r, 0.27 r after 600; the mean over 32768 elements: 0.0015."""
    from clt_training_amd import hip_ops as ops

    n = 32768
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    y = torch.linspace(100, 440, n, device="cuda")[torch.randperm(n, generator=torch.Generator().manual_seed(0)).cuda()]
    v = (y.to(torch.float8_e4m3fn), torch.full((n // 128,), 120, dtype=torch.uint8, device="cuda"))
    m = (torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n // 128, dtype=torch.uint8, device="cuda"))
    start = decode(*v).mean()
    for t in range(1, 601):
        ops.adamw_step([p], [g], [m], [v], step=t, seed=3)
    assert abs(float(decode(*v).mean() / start) / B2**300 - 1) < 6 * 0.0015
    assert (p == 0).all()


@pytest.mark.gpu
def test_more_than_2_to_32_elements():
    """Offsets past 32 bits in every array: slices of the result against the oracle, with the random bits of their elements."""
    from clt_training_amd import hip_ops as ops

    n = 2**32 + 1000
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = ((torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(-(-n // 128), dtype=torch.uint8, device="cuda")) for _ in range(2))
    spots = [slice(0, 256), slice(2**31 - 128, 2**31 + 128), slice(2**32 - 256, 2**32 + 256), slice(n - 232, n)]
    for k, s in enumerate(spots):
        x = make((s.stop - s.start,), torch.bfloat16, torch.bfloat16, False, 40 + k)
        p[s], g[s] = x[0], x[1]
    before = [(p[s].clone(), g[s].clone()) for s in spots]
    ops.adamw_step([p], [g], [m], [v], step=1, lr=LR, weight_decay=WD, seed=9)
    for (p0, g0), s in zip(before, spots):
        idx = torch.arange(s.start, s.stop, device="cuda")
        gd = g0.double()
        m_new, r_new = (1 - B1) * gd, math.sqrt(1 - B2) * gd.abs()
        D = LR * gd / (gd.abs() + EPS)
        want = p0.double() * (1 - LR * WD) - D
        room = U * (3 * p0.double().abs() + 40 * D.abs())
        assert ((p[s].double() - want).abs() <= room + 2.0**-8 * (want.abs() + room)).all()
        lo, hi = chances(9, 0, 1, idx)
        blk = slice(s.start // 128, -(-s.stop // 128))
        check_8bit(m[0][s], m[1][blk], m_new, lo, False)
        check_8bit(v[0][s], v[1][blk], r_new, hi, True)
    assert int((p != 0).sum()) <= sum(s.stop - s.start for s in spots)


@pytest.mark.gpu
def test_refuses_what_shares_memory():
    from clt_training_amd import hip_ops as ops

    p, g, m, v = make((300,), torch.float32, torch.float32, False, 1)
    before = p.clone()
    part = lambda t, k: t[k:k + 100]  # noqa: E731
    with pytest.raises(ValueError, match="share memory"):  # (two parameters that overlap in part)
        ops.adamw_step([part(p, 0), part(p, 99)], [part(g, 0), part(g, 100)], [part(m, 0), part(m, 100)], [part(v, 0), part(v, 100)], step=1)
    with pytest.raises(ValueError, match="share memory"):  # (a gradient that is another tensor's moment)
        ops.adamw_step([part(p, 0), part(p, 100)], [part(g, 0), part(m, 50)], [part(m, 0), part(m, 100)], [part(v, 0), part(v, 100)], step=1)
    q, h, n, w = make((300,), torch.float32, torch.float32, True, 2)
    with pytest.raises(ValueError, match="share memory"):  # (one array of scales for both moments)
        ops.adamw_step([q], [h], [n], [(w[0], n[1])], step=1)
    assert torch.equal(p, before)
    ops.adamw_step([part(p, 0), part(p, 100)], [part(g, 0), part(g, 0)], [part(m, 0), part(m, 100)], [part(v, 0), part(v, 100)], step=1)  # (shared gradients are fine)


@pytest.mark.gpu
def test_streams_refusals_and_repeats():
    from clt_training_amd import hip_ops as ops
    from clt_training_amd.adam import AdamW

    a, b = (make((5000,), torch.bfloat16, torch.bfloat16, True, 1) for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adamw_step([a[0]], [a[1]], [a[2]], [a[3]], step=5, seed=2)
    torch.cuda.current_stream().wait_stream(s)
    ops.adamw_step([b[0]], [b[1]], [b[2]], [b[3]], step=5, seed=2)
    for x, y in ((a[0], b[0]), *zip(a[2], b[2]), *zip(a[3], b[3])):
        assert torch.equal(x, y)
    c = make((5000,), torch.bfloat16, torch.bfloat16, True, 1)
    ops.adamw_step([c[0]], [c[1]], [c[2]], [c[3]], step=5, seed=3)
    assert torch.equal(c[0], b[0]) and not torch.equal(c[2][0], b[2][0])  # another seed: other roundings of the moments only
    p, g, m, v = make((64,), torch.float32, torch.float32, False, 1)
    q, h, n, w = make((64,), torch.float32, torch.float32, False, 2)
    ok = dict(step=1)
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p, p], [g, h], [m, n], [v, w], **ok)
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p, q], [g, h], [m, n], [v, v], **ok)
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p], [g], [m], [m], **ok)
    with pytest.raises(TypeError):
        ops.adamw_step([p.half()], [g], [m], [v], **ok)
    with pytest.raises(TypeError):
        ops.adamw_step([p], [g], [m.bfloat16()], [v.bfloat16()], **ok)
    with pytest.raises(ValueError):
        ops.adamw_step([p], [g[:32]], [m], [v], **ok)
    with pytest.raises(ValueError):
        ops.adamw_step([p.expand(2, 64)], [g.expand(2, 64)], [m.expand(2, 64)], [v.expand(2, 64)], **ok)
    with pytest.raises(ValueError, match="both"):
        ops.adamw_step([p], [g], [m], [(v, v)], **ok)
    with pytest.raises(ValueError):
        ops.adamw_step([p], [g], [(m.to(torch.uint8), m[:2].to(torch.uint8))], [(v.to(torch.uint8), v[:1].to(torch.uint8))], **ok)
    with pytest.raises(ValueError, match="per tensor"):
        ops.adamw_step([p], [g], [m], [v], lr=[0.1, 0.2], **ok)
    with pytest.raises(RuntimeError, match="status -1"):
        ops.adamw_step([p], [g], [m], [v], step=0)
    x = torch.nn.Parameter(p.clone())
    x.grad = g.clone()
    opt = AdamW([x])
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(4, device="cuda")
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        with pytest.raises(RuntimeError, match="captured"):
            ops.adamw_step([p], [g], [m], [v], **ok)
    assert opt._step == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_steps(bits):
    """Ten steps, a parameter without a gradient among them: with 32 bits against torch.optim.AdamW in 64 bits, with 8 against
    adamw_step on states of its own (the same bits); a fresh optimizer that loads the state goes on with the same bits.
    Room with 32 bits: ten steps, each off by 8 u of a parameter of size <= 8 (an update of 1e-2 adds less)."""
    import io

    from clt_training_amd import hip_ops as ops
    from clt_training_amd.adam import AdamW

    gen = torch.Generator().manual_seed(0)
    shapes = [(70, 65), (300,), (9,)]
    start = [torch.randn(s, generator=gen) for s in shapes]
    grads = [[torch.randn(s, generator=gen) * 10.0 ** (i - 2) for i, s in enumerate(shapes)] for _ in range(10)]

    def groups(ps):
        return [dict(params=ps[:1], lr=torch.tensor(1e-2)), dict(params=ps[1:], lr=3e-3, weight_decay=0.1)]

    def optimizer(ps):
        opt = AdamW(groups(ps), weight_decay=0.01, state_bits=bits, seed=11)
        extra = torch.nn.Parameter(torch.ones(3, device="cuda"))
        opt.add_param_group(dict(params=[extra]))
        return opt, extra

    mine = [torch.nn.Parameter(p.cuda()) for p in start]
    opt, extra = optimizer(mine)
    if bits == 32:
        ref = [torch.nn.Parameter(p.double()) for p in start]
        ropt = torch.optim.AdamW(groups(ref), weight_decay=0.01)
    else:
        ref = [p.cuda() for p in start]
        zeros = lambda n: (torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(-(-n // 128), dtype=torch.uint8, device="cuda"))  # noqa: E731
        moments = [[zeros(4550), torch.zeros(300, device="cuda"), torch.zeros(9, device="cuda")] for _ in range(2)]
    for k, gs in enumerate(grads):
        for p, g in zip(mine, gs):
            p.grad = g.cuda()
        if bits == 32:
            for p, g in zip(ref, gs):
                p.grad = g.double()
            ropt.step()
        else:
            ops.adamw_step(ref, [g.cuda() for g in gs], *moments, step=k + 1, lr=[float(torch.tensor(1e-2)), 3e-3, 3e-3],
                           weight_decay=[0.01, 0.1, 0.1], seed=11)
        if k == 6:  # through a file
            buf = io.BytesIO()
            torch.save(opt.state_dict(), buf)
            buf.seek(0)
            twin = [torch.nn.Parameter(p.detach().clone()) for p in mine]
            topt, _ = optimizer(twin)
            topt.load_state_dict(torch.load(buf, weights_only=True))
        opt.step()
        if k >= 6:
            for p, g in zip(twin, gs):
                p.grad = g.cuda()
            topt.step()
    for a, b in zip(mine, twin):
        assert torch.equal(a, b)
    assert (extra == 1).all()
    kinds = {k for st in opt.state.values() for k in st}
    assert ("rms_codes" in kinds) == (bits == 8) and "exp_avg" in kinds
    for a, b in zip(mine, ref):
        if bits == 32:
            assert float((a.detach().cpu().double() - b.detach()).abs().max()) < 10 * 8 * U * 8
        else:
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_trainer_saves_and_resumes(optimizer, tmp_path):
    """A run interrupted by a checkpoint ends with the parameters of the uninterrupted one, bit for bit."""
    from clt_training_amd import SparseCoderConfig, TrainConfig, Trainer

    def batches():
        g = torch.Generator().manual_seed(4)
        return [{h: (torch.randn(64, 64, generator=g).cuda(), torch.randn(64, 64, generator=g).cuda()) for h in ("a", "b")} for _ in range(6)]

    def trainer():
        cfg = TrainConfig(sae=SparseCoderConfig(dtype="bfloat16", k=4, expansion_factor=4, transcode=True), hookpoints=["a", "b"], cross_layer=2,
                          optimizer=optimizer, lr=1e-2, lr_warmup_steps=1)
        return Trainer(cfg, batches())

    whole = trainer()
    for b in batches():
        whole.step(b)
    first = trainer()
    for b in batches()[:3]:
        first.step(b)
    first.save(tmp_path)
    second = trainer().load_state(tmp_path)
    for b in batches()[3:]:
        second.step(b)
    for (n, p), (_, q) in zip(((n, p) for s in whole.saes.values() for n, p in s.named_parameters()), ((n, p) for s in second.saes.values() for n, p in s.named_parameters())):
        assert torch.equal(p, q), n


@pytest.mark.gpu
def test_late_parameters_against_torch():
    """Parameters whose gradients come and go, against torch.optim.AdamW in 64 bits.  Room: as in test_optimizer_steps, twelve
    steps off by 8 u of a parameter of size <= 8 each."""
    from clt_training_amd.adam import AdamW

    gen = torch.Generator().manual_seed(2)
    start = [torch.randn(n, generator=gen) for n in (300, 40, 7)]
    mine, ref = [torch.nn.Parameter(p.cuda()) for p in start], [torch.nn.Parameter(p.double()) for p in start]
    opt, ropt = AdamW(mine, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    for k in range(12):
        for i, (p, q) in enumerate(zip(mine, ref)):
            g = torch.randn(p.shape, generator=gen) if k >= 5 * i and (k + i) % 4 else None
            p.grad, q.grad = (None, None) if g is None else (g.cuda(), g.double())
        opt.step()
        ropt.step()
    for p, q in zip(mine, ref):
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) < 12 * 8 * U * 8


@pytest.mark.gpu
def test_subnormal_second_moments_32():
    """v below 2^-126 has a root of its own, also with eps = 0.  b2 v is rounded to fp32's least steps, so the root's argument is
    v as the call left it; from there on the module's 20 u of the update."""
    from clt_training_amd import hip_ops as ops

    n = 4096
    gen = torch.Generator().manual_seed(1)
    v = (torch.randint(2, 2**23, (n,), generator=gen) >> torch.randint(0, 21, (n,), generator=gen)).clamp(min=2).to(torch.int32).view(torch.float32)
    assert float(v.min()) > 0 and float(v.max()) < 2.0**-126
    v[1::4] = 2.0**-126 * (1 + torch.rand(v[1::4].shape, generator=gen))  # (normal neighbours)
    m = torch.randn(n, generator=gen) * torch.sqrt(v.double()).float()
    p, v, m = torch.zeros(n, device="cuda"), v.cuda(), m.cuda()
    before = m.clone()
    ops.adamw_step([p], [torch.zeros(n, device="cuda")], [m], [v], step=10, lr=1.0, betas=(B1, B2), eps=0.0, weight_decay=0.0)
    assert bool((v > 0).all())
    want = -1 / (1 - B1**10) * B1 * before.double() * math.sqrt(1 - B2**10) / torch.sqrt(v.double())
    room = U * 20 * want.abs() + 3 * U * want.abs() + 2.0**-149  # (3 u: m', whose gradient is 0)
    assert ((p.double() - want).abs() <= room).all()


@pytest.mark.gpu
def test_subnormal_second_moments_8():
    """The stored root of a subnormal v: r > 0 stays > 0 wherever v = b2 r^2, formed in fp32, is."""
    from clt_training_amd import hip_ops as ops

    n = 126 * 128
    codes = (torch.arange(n) % 126 + 1).to(torch.uint8)  # every positive value of e4m3
    scale = torch.arange(126) % 14 + 127 - 80  # r^2 from below fp32's least step to normal numbers
    r = codes.view(torch.float8_e4m3fn).float() * torch.exp2((scale - 127).double()).float().repeat_interleave(128)
    v_new = r * r * torch.tensor(B2, dtype=torch.float32)
    assert bool(((v_new > 0) & (v_new < 2.0**-126)).any()) and bool((v_new == 0).any()) and bool((v_new > 2.0**-126).any())
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m = (torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(126, dtype=torch.uint8, device="cuda"))
    second = (codes.cuda(), scale.to(torch.uint8).cuda())
    ops.adamw_step([p], [g], [m], [second], step=4, betas=(B1, B2), seed=8)
    _, hi = chances(8, 0, 4, torch.arange(n, device="cuda"))
    check_8bit(*second, torch.sqrt(v_new.double()).cuda(), hi, True)
    assert bool((p == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_autograd_sees_that_a_step_changed_its_tensors(eight):
    """A parameter that changed between forward and backward is an error, as with torch's optimizers; a refused call changes
    nothing; tensors of inference mode, which keep no count, are taken."""
    from clt_training_amd import hip_ops as ops

    p, g, m, v = make((256,), torch.float32, torch.float32, eight, 1)
    moments = [*m, *v] if eight else [m, v]
    x = torch.ones(256, device="cuda", requires_grad=True)
    y = (x * p).sum()
    versions = [t._version for t in (p, g, *moments)]
    with pytest.raises(RuntimeError):
        ops.adamw_step([p], [g], [m], [v], step=0)
    assert [t._version for t in (p, g, *moments)] == versions
    ops.adamw_step([p], [g], [m], [v], step=1)
    assert [t._version - w for t, w in zip((p, g, *moments), versions)] == [1, 0] + [1] * len(moments)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        p, g, m, v = make((256,), torch.float32, torch.float32, eight, 1)
        ops.adamw_step([p], [g], [m], [v], step=1)
    ops.adamw_step([p], [g], [m], [v], step=2)
