"""AdamW with both moments in 8 bits: the code, the step, the optimizer class.

The moments' arithmetic is that of the plain statement, every operation rounded by itself: equal bits are asked for.  A parameter's update has an
approximate root and quotient, 2 units each, and the roundings of four operations, 2^-20 of it in all, and the sum is rounded twice, 2^-23 of the
parameter; a bf16 shadow may then round to either side.  Against 64 bits: a moment
kept is off by less than one step of its code (an eighth of |x| a / TOP + FIRST, at most) and 2^-20 for the fp32 arithmetic before it."""

import copy

import pytest
import torch

from torchure_b200 import ops
from torchure_b200.ops import multi_tensor, oracle
from torchure_b200.optim.adamw import AdamW
from torchure_b200.optim.builder import build_optimizer

GPU = pytest.param("cuda", marks=pytest.mark.gpu)
FIRST, TOP = {True: 2.0 ** -15, False: 2.0 ** -31}, {True: 1.875 - 2.0 ** -15, False: 1.875}
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def code_values(signed):
    """What each code stands for, over the scale, from the format's description."""
    out = []
    for code in range(256):
        size = code & 127 if signed else code
        y = 2.0 ** (size // 8 - (15 if signed else 31)) * (1 + size % 8 / 8) - FIRST[signed]
        out.append(-y if signed and code >= 128 else y)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("signed", [True, False])
def test_codes_stand_for_what_the_format_says(signed):
    codes = torch.arange(256).to(torch.uint8)
    scales = torch.tensor([0.5, 3.0])
    want = code_values(signed) * torch.tensor([0.5, 3.0], dtype=torch.float64).repeat_interleave(128)
    got = oracle.state8_decode(codes, scales, signed).double()
    assert ((got - want).abs() <= 2.0 ** -23 * want.abs()).all()          # one product in fp32
    assert (code_values(signed)[:128].diff() > 0).all() and float(code_values(signed).max().float()) == TOP[signed]
    # what a code stands for goes to that code again, whatever the random bits: but for a unit of fp32, in steps of 2^20 units
    block = code_values(signed).float() * (0.7 / TOP[signed])
    block = torch.cat([block[:128], block[127:128] if signed else block[255:256]])[-128:] if signed else block
    parts = block.view(-1, 128)
    for part in parts:
        x = torch.cat([part[:127], torch.tensor([0.7])])                  # the block's largest sets the scale
        again = oracle.state8_decode(*oracle.state8_encode(x, torch.full((128,), 32768), signed), signed)
        assert ((again - x).abs() <= 2.0 ** -20 * x.abs()).all()


@pytest.mark.parametrize("signed", [True, False])
def test_rounding_keeps_the_mean(signed):
    """Over all random bits the mean of what is kept is the value, to a unit of the 2^16 bits; to the nearest, at most half a step off."""
    x = torch.tensor([0.9, 0.013, 3e-4, 1e-6, 0.0, 0.33, -0.2 if signed else 0.2])
    rows = torch.cat([torch.ones(1), x, torch.zeros(120)])
    r = torch.arange(0, 65536, 16) + 8                                    # 4096 even places
    kept = torch.stack([oracle.state8_decode(*oracle.state8_encode(rows, torch.full((128,), int(v)), signed), signed)[1:8] for v in r]).double()
    y = x.abs().double() * TOP[signed] + FIRST[signed]
    step = torch.exp2(torch.floor(torch.log2(y)) - 3) / TOP[signed]
    assert ((kept.mean(0) - x.double()).abs() <= step * 2.0 ** -11 + 2.0 ** -22).all()      # 4096 of 65536 places: half a place is 2^-13
    assert ((kept - x.double()).abs() < step * (1 + 2.0 ** -15) + 2.0 ** -22).all()
    near = oracle.state8_decode(*oracle.state8_encode(rows, torch.full((128,), 32768), signed), signed)[1:8].double()
    assert ((near - x.double()).abs() <= step * 0.5 + 2.0 ** -20).all()


def test_small_blocks_and_blocks_that_are_not_finite():
    for signed in (True, False):
        x = torch.rand(5 * 128)
        x[0:128] = 0
        x[128] = float("nan")
        x[256] = float("inf")
        x[384:512] *= 2.0 ** -101
        x[512:] *= 2.0 ** -90
        codes, scales = oracle.state8_encode(x, torch.zeros(640, dtype=torch.int64), signed)
        y = oracle.state8_decode(codes, scales, signed).view(5, 128)
        assert (y[0] == 0).all() and torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and (y[3] == 0).all()
        assert ((y[4] - x[512:]).abs() <= x[512:] * 0.13 + 2.0 ** -100).all()
    # next to a large one a second moment is never rounded to nothing
    v = torch.full((128,), 1e-30)
    v[0], v[1] = 1.0, 0.0
    codes, _ = oracle.state8_encode(v, torch.zeros(128, dtype=torch.int64), False)
    assert codes[1] == 0 and (codes[2:] == 1).all()


def near(got, want, before, steps=1):
    """Parameters after so many steps whose updates are at most what ``want`` is away from ``before`` and the decay together."""
    got, want, before = (t.detach().double().cpu() for t in (got, want, before))
    update = (want - before).abs() + steps * 1e-3 * before.abs() + steps * 0.2          # (single updates: at most some 10 lr)
    return bool(((got - want).abs() <= steps * (2.0 ** -23 * (before.abs() + 0.2) + 2.0 ** -20 * update)).all())


SHAPES = [(1,), (127,), (3, 43), (128,), (129,), (7, 1000), (16384,), (16385,), (5, 3333), (40000,)]


def problem(seed, device="cpu", half=False, shadow=True, steps_before=3):
    """Parameters of many sizes with moments that have seen a few steps."""
    g = torch.Generator().manual_seed(seed)
    s = dict(params=[], grads=[], ms=[], mscales=[], vs=[], vscales=[], shadows=[])
    for i, shape in enumerate(SHAPES):
        strength = torch.exp(torch.randn(shape[0], *[1] * (len(shape) - 1), generator=g)) * 1e-2
        s["params"].append(torch.randn(shape, generator=g))
        grad = torch.randn(shape, generator=g) * strength
        s["grads"].append(grad.bfloat16() if half and i % 2 else grad)
        s["shadows"].append(s["params"][-1].bfloat16() if shadow and i % 3 else None)
        for name, x, signed in (("m", torch.randn(shape, generator=g) * strength, True), ("v", torch.rand(shape, generator=g) * strength ** 2, False)):
            codes, scales = oracle.state8_encode(x, torch.randint(0, 65536, (x.numel(),), generator=g), signed)
            s[name + "s"].append(codes)
            s[name + "scales"].append(scales)
    return {n: [None if t is None else t.to(device) for t in ts] for n, ts in s.items()}


def step(s, f, **kw):
    f(s["params"], s["grads"], s["ms"], s["mscales"], s["vs"], s["vscales"], s["shadows"], **{**HYPER, **kw})


def plain(params, grads, ms, msc, vs, vsc, shadows, lr, beta1, beta2, eps, weight_decay, step, **kw):
    oracle.adamw8(params, grads, ms, msc, vs, vsc, shadows, lr, beta1, beta2, eps, weight_decay, step, **kw)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_step_against_the_definition(device):
    s = problem(1, device)
    before = {n: [None if t is None else t.clone() for t in ts] for n, ts in s.items()}
    step(s, multi_tensor.adamw8_step, step=7, seed=5)
    for i, p in enumerate(before["params"]):
        g = before["grads"][i].double()
        m = 0.9 * oracle.state8_decode(before["ms"][i], before["mscales"][i], True).double() + 0.1 * g
        v = 0.95 * oracle.state8_decode(before["vs"][i], before["vscales"][i], False).double() + 0.05 * g * g
        want = p.double() * (1 - 1e-3) - 1e-2 * (m / (1 - 0.9 ** 7)) / ((v / (1 - 0.95 ** 7)).sqrt() + 1e-8)
        # ten operations of 2^-24 on an update of at most a few times lr, two on the parameter
        assert ((s["params"][i].double() - want).abs() <= 2.0 ** -20 * (p.double().abs() + 0.1)).all()
        if s["shadows"][i] is not None:
            assert torch.equal(s["shadows"][i], s["params"][i].bfloat16())
        for x, codes, scales, signed in ((m, s["ms"][i], s["mscales"][i], True), (v, s["vs"][i], s["vscales"][i], False)):
            kept = oracle.state8_decode(codes, scales, signed).double()
            flat = torch.nn.functional.pad(x.abs().reshape(-1), (0, -x.numel() % 128)).view(-1, 128)
            scale = (flat.amax(1, keepdim=True) / TOP[signed]).expand_as(flat).reshape(-1)[:x.numel()].view(x.shape)
            bound = (x.abs() + FIRST[signed] * scale) * 0.125 + 2.0 ** -20 * x.abs()
            assert ((kept - x).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shadow", [False, True])
@pytest.mark.parametrize("clip", [None, 0.37])
@pytest.mark.parametrize("maximize", [False, True])
def test_kernel_has_the_plain_statements_bits(half, shadow, clip, maximize):
    a, b = problem(2, "cpu", half, shadow), problem(2, "cuda", half, shadow)
    start = [p.clone() for p in a["params"]]
    for t in (1, 2, 1000):
        gs = None if clip is None else torch.tensor(clip)
        step(a, plain, step=t, seed=9, grad_scale=gs, maximize=maximize)
        step(b, multi_tensor.adamw8_step, step=t, seed=9, grad_scale=None if gs is None else gs.cuda(), maximize=maximize)
    for name in ("grads", "ms", "mscales", "vs", "vscales"):
        assert all(torch.equal(x, y.cpu()) for x, y in zip(a[name], b[name])), name
    assert all(near(y, x, s, 3) for x, y, s in zip(a["params"], b["params"], start))
    assert all(x is None or torch.equal(x, p.bfloat16()) for x, p in zip(b["shadows"], b["params"]))
    for signed, codes, scales in ((True, "ms", "mscales"), (False, "vs", "vscales")):
        for dtype in (torch.float32, torch.bfloat16):
            got = multi_tensor.state8_values(b[codes], b[scales], signed, dtype)
            want = multi_tensor.state8_values(a[codes], a[scales], signed, dtype)
            assert all(torch.equal(x.cpu(), y) and x.shape == y.shape for x, y in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_any_alignment(shift):
    """Gradients, parameters, codes and shadows that begin anywhere in a buffer; what lies around them stays."""
    a, b = problem(3, "cpu"), problem(3, "cuda")

    def moved(t):
        if t is None:
            return None
        room = torch.full((t.numel() + 8,), 77, dtype=t.dtype, device=t.device)
        room[shift:shift + t.numel()] = t.reshape(-1)
        return room[shift:shift + t.numel()].view(t.shape)

    b = {n: [moved(t) for t in ts] for n, ts in b.items()}
    c = problem(3, "cuda")
    step(a, plain, step=4, seed=1)
    step(b, multi_tensor.adamw8_step, step=4, seed=1)
    step(c, multi_tensor.adamw8_step, step=4, seed=1)
    for name in a:
        for w, x, y in zip(a[name], c[name], b[name]):
            if x is not None:
                assert torch.equal(x, y), name
                assert name in ("params", "shadows") or torch.equal(w, y.cpu()), name
                room = y._base if y._base is not None else y
                assert int((room[:shift] == 77).sum()) == shift and int((room[shift + y.numel():] == 77).sum()) == 8 - shift
    values = multi_tensor.state8_values(b["ms"], b["mscales"], True)
    assert all(torch.equal(v.cpu(), oracle.state8_decode(c, s, True)) for v, c, s in zip(values, a["ms"], a["mscales"]))


@pytest.mark.gpu
def test_not_finite_gradients_stay_in_their_block():
    s = problem(4, "cuda")
    s["grads"][9][200], s["grads"][9][1000] = float("nan"), float("inf")
    step(s, multi_tensor.adamw8_step, step=2)
    p, m, v = s["params"][9], *(multi_tensor.state8_values([s[c][9]], [s[k][9]], sg)[0] for c, k, sg in (("ms", "mscales", True), ("vs", "vscales", False)))
    bad = torch.zeros(40000, dtype=torch.bool, device="cuda")
    bad[128:256] = bad[896:1024] = True
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
    assert torch.isnan(p).sum() == 2 and torch.isnan(p[200]) and torch.isnan(p[1000])


@pytest.mark.gpu
def test_a_second_moment_that_overflows():
    """The step itself divides by infinity; the block's second moment is NaN from then on, and the next step's parameters say so."""
    a, b = problem(8, "cpu"), problem(8, "cuda")
    for s in (a, b):
        s["grads"][8][0, 5] = 1e25
    for t in (1, 2):
        step(a, plain, step=t)
        step(b, multi_tensor.adamw8_step, step=t)
        bad = torch.isnan(a["params"][8])
        assert torch.equal(bad, torch.isnan(b["params"][8]).cpu()) and int(bad.sum()) == (0 if t == 1 else 128)
        assert torch.isfinite(b["params"][8][~bad.cuda()]).all()
        for name in ("ms", "vs"):
            assert torch.equal(a[name][8], b[name][8].cpu())


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("eps", [0.0, 1e-8])
def test_zero_and_tiny_gradients(device, eps):
    """Nothing where nothing came; with eps 0 too, where 0 / 0 would be."""
    p = torch.linspace(-1, 1, 1000)
    for value in (0.0, 1e-30, 1e-20):
        s = dict(params=[p.to(device, copy=True)], grads=[torch.zeros(1000, device=device)], ms=[torch.zeros(1000, dtype=torch.uint8, device=device)],
                 vs=[torch.zeros(1000, dtype=torch.uint8, device=device)], mscales=[torch.zeros(8, device=device)],
                 vscales=[torch.zeros(8, device=device)], shadows=[None])
        s["grads"][0][:500] = value
        for t in (1, 2):
            step(s, multi_tensor.adamw8_step, step=t, eps=eps)
        got = s["params"][0].cpu()
        assert torch.isfinite(got).all()
        assert torch.allclose(got[500:], p[500:] * (1 - 1e-3) ** 2, rtol=1e-6, atol=0)
        # at most the two updates of lr, whatever came
        assert ((got[:500] - p[:500] * (1 - 1e-3) ** 2).abs() <= 2.1e-2).all()


@pytest.mark.gpu
def test_a_tensor_beyond_32_bits():
    """Indexes and random bits of the last elements, as the plain statement has them."""
    n = (1 << 32) + 300
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    m, v = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    ms, vs = torch.zeros(-(-n // 128), device="cuda"), torch.zeros(-(-n // 128), device="cuda")
    lo = (1 << 32) - 256
    tail = torch.randn(n - lo, generator=torch.Generator().manual_seed(0)).bfloat16()
    g[lo:] = tail.cuda()
    multi_tensor.adamw8_step([p], [g], [m], [ms], [v], [vs], [None], step=3, seed=2, **HYPER)
    assert int(torch.count_nonzero(p[:lo:4097])) == 0 and int(torch.count_nonzero(m[:lo:4097])) == 0
    key = oracle.state8_key(2, 3)
    i = torch.arange(lo, n)
    bits = oracle._mix32((i & 0xFFFFFFFF) ^ oracle._mix32((key + 0xC2B2AE35 * (i >> 32)) & 0xFFFFFFFF))
    for x, r, codes, scales, signed in ((tail.float() * (1.0 - 0.9), bits & 0xFFFF, m, ms, True),
                                        ((tail.float() * (1.0 - 0.95)) * tail.float(), bits >> 16, v, vs, False)):
        want, want_scales = oracle.state8_encode(x, r, signed)
        assert torch.equal(codes[lo:].cpu(), want) and torch.equal(scales[lo // 128:].cpu(), want_scales)
    del p, g, m, v, ms, vs
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_refusals_of_the_step():
    def refused(name, make):
        s = problem(5, "cuda")
        s[name][3] = make(s[name][3])
        with pytest.raises((ValueError, TypeError)):
            step(s, multi_tensor.adamw8_step, step=1)

    refused("params", lambda t: t.bfloat16())
    refused("grads", lambda t: t.half())
    refused("grads", lambda t: t[:100])
    refused("grads", lambda t: t.cpu())
    refused("grads", lambda t: torch.stack([t, t], 1)[:, 0])
    refused("ms", lambda t: t.to(torch.int8))
    refused("vs", lambda t: t[1:])
    refused("mscales", lambda t: torch.cat([t, t]))
    refused("vscales", lambda t: t.double())
    refused("shadows", lambda t: torch.zeros(128, device="cuda"))
    s = problem(5, "cuda")
    s["shadows"] = s["shadows"][:-1]
    with pytest.raises(ValueError):
        step(s, multi_tensor.adamw8_step, step=1)
    with pytest.raises(ValueError):
        step(problem(5, "cuda"), multi_tensor.adamw8_step, step=1, grad_scale=torch.tensor(1.0))
    for hyper in (torch.zeros(8, device="cuda")[::2], torch.zeros(3, device="cuda"), torch.zeros(4)):
        with pytest.raises(ValueError):
            step(problem(5, "cuda"), multi_tensor.adamw8_step, step=1, hyper=hyper)
    with pytest.raises(TypeError):
        multi_tensor.state8_values(s["ms"], s["mscales"], True, torch.float16)
    with pytest.raises(ValueError):
        multi_tensor.state8_values(s["ms"], s["mscales"][1:], True)
    assert multi_tensor.state8_values([], [], True) == []
    multi_tensor.adamw8_step([], [], [], [], [], [], [], step=1, **HYPER)


# ---- the optimizer ----------------------------------------------------------------------------------
def train(device, steps=6, bits=8, seed=0, opt_seed=3, opt=None, params=None, first=0, shadow=False):
    g = torch.Generator().manual_seed(seed)
    made = [torch.randn(37, 50, generator=g), torch.randn(300, generator=g), torch.randn(2, 3, 129, generator=g)]
    if params is None:
        params = [torch.nn.Parameter(t.to(device)) for t in made]
    if opt is None:
        opt = build_optimizer(None, "adamw", dict(lr=1e-2, weight_decay=0.1, betas=[0.9, 0.95], fused=True, state_bits=bits,
                                                  **({"rounding_seed": opt_seed} if bits == 8 else {})), params=params)
    for t in range(first, first + steps):
        g = torch.Generator().manual_seed(100 + t)
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(device)
        if device == "cuda" and t % 2:
            opt.set_grad_scale(torch.tensor(0.5, device=device))
        elif t % 2:
            opt.set_grad_scale(torch.tensor(0.5))
        opt.step()
    return params, opt


@pytest.mark.gpu
def test_optimizer_on_the_gpu_equals_the_cpus():
    (a, oa), (b, ob) = train("cpu"), train("cuda")
    start, _ = train("cpu", 0)
    for p, q, s in zip(a, b, start):
        assert near(q, p, s, 6)
        assert all(torch.equal(oa.state[p][n], ob.state[q][n].cpu()) for n in oa.state[p])


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_optimizer_follows_the_32_bit_one(device):
    """Ten steps: the second moment is off by its code's steps (each at most an eighth, a twentieth of which is new every step), so an update by
    at most a half; the sum of updates of either is at most 10 lr (1 + wd) + what the first moment's code adds, an eighth of lr each."""
    (a, _), (b, _) = train(device, 10, 8), train(device, 10, 32)
    start, _ = train(device, 0, 32)
    for p, q, s in zip(a, b, start):
        assert float((p - q).detach().norm()) < 0.25 * float((q - s).detach().norm())


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_state_dicts_resume_bit_for_bit_and_convert(device, tmp_path):
    params, opt = train(device, 4)
    torch.save(opt.state_dict(), tmp_path / "o.pt")
    kept = [p.detach().clone() for p in params]
    train(device, 3, opt=opt, params=params, first=4)
    again = [torch.nn.Parameter(t.clone()) for t in kept]
    fresh = build_optimizer(None, "adamw", dict(lr=1e-2, weight_decay=0.1, betas=[0.9, 0.95], fused=True, state_bits=8, rounding_seed=3),
                            params=again)
    fresh.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    assert all(fresh.state[p]["exp_avg"].dtype == torch.uint8 and fresh.state[p]["exp_avg"].device == p.device for p in again)
    train(device, 3, opt=fresh, params=again, first=4)
    assert all(torch.equal(p, q) for p, q in zip(params, again))
    # to 32 bits: the values; back: the same codes
    wide = AdamW([torch.nn.Parameter(t.clone()) for t in kept], fused=True)
    sd = torch.load(tmp_path / "o.pt", weights_only=True)
    one = copy.deepcopy(sd)
    one["param_groups"] = [dict(one["param_groups"][0], params=[0, 1, 2])]
    wide.load_state_dict(one)
    for i, st in sd["state"].items():
        got = wide.state[wide.param_groups[0]["params"][i]]
        assert set(got) == {"step", "exp_avg", "exp_avg_sq"}
        assert torch.equal(got["exp_avg"], oracle.state8_decode(st["exp_avg"], st["exp_avg_scale"], True).to(got["exp_avg"].device))
    back = AdamW([torch.nn.Parameter(t.clone()) for t in kept], fused=True, state_bits=8)
    back.load_state_dict(wide.state_dict())
    for i, st in sd["state"].items():
        got = back.state[back.param_groups[0]["params"][i]]
        for key, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            x = oracle.state8_decode(st[key], st[key + "_scale"], signed)
            y = oracle.state8_decode(got[key], got[key + "_scale"], signed).to(x.device)
            assert ((x - y).abs() <= 2.0 ** -20 * x.abs()).all()


def test_a_state_dict_for_parameters_in_16_bits():
    """An optimizer without 8-bit moments may have such parameters: the moments come in their type, rounded once, and the next step runs."""
    _, opt = train("cpu", 4)
    sd = copy.deepcopy(opt.state_dict())
    sd["param_groups"] = [dict(sd["param_groups"][0], params=[0, 1, 2])]
    half = [torch.nn.Parameter(p.detach().bfloat16()) for g in opt.param_groups for p in g["params"]]
    wide = AdamW(half)
    wide.load_state_dict(sd)
    for i, p in enumerate(half):
        st = sd["state"][i]
        assert st["exp_avg"].dtype == torch.uint8      # (the caller's stays)
        for key, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            assert torch.equal(wide.state[p][key], oracle.state8_decode(st[key], st[key + "_scale"], signed).bfloat16())
        p.grad = torch.ones_like(p)
    wide.step()


def test_a_refused_group_is_not_kept():
    opt = AdamW([torch.nn.Parameter(torch.zeros(4))], state_bits=8)
    with pytest.raises(TypeError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16))]})
    assert len(opt.param_groups) == 1


def test_refusals_of_the_optimizer():
    p = torch.nn.Parameter(torch.randn(4, 4))
    for kw in (dict(state_bits=16), dict(state_bits=8, amsgrad=True)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.randn(4, 4).bfloat16())], state_bits=8)
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.randn(4, 6).t())], state_bits=8)
    with pytest.raises(ValueError):
        multi_tensor.state8_values([torch.zeros(3, dtype=torch.uint8)], [], True)


@pytest.mark.gpu
def test_replayed_steps_equal_eager_ones():
    """A captured step reads its scalars and the key of its random bits from device memory; another captured optimizer of the same sizes, and
    eager steps between the replays, have tables of their own."""
    g = torch.Generator().manual_seed(0)
    start = [torch.randn(64, 300, generator=g), torch.randn(77, generator=g)]
    grads = [[torch.randn(t.shape, generator=g) for t in start] for _ in range(5)]

    def make():
        params = [torch.nn.Parameter(t.cuda()) for t in start]
        opt = build_optimizer(None, "adamw", dict(lr=1e-2, weight_decay=0.1, betas=[0.9, 0.95], fused=True, state_bits=8), params=params)
        for p in params:
            p.grad = torch.zeros_like(p)
        return params, opt

    eager, eo = make()
    graphs = []
    for _ in range(2):
        params, opt = make()
        opt.enable_device_hyper()
        for p, q in zip(params, grads[0]):
            p.grad.copy_(q)
        opt.step()
        snap = opt.host_state()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        opt.restore_host_state(snap)
        graphs.append((params, opt, graph))
    for t in range(5):
        for p, q in zip(eager, grads[t]):
            p.grad.copy_(q)
        eo.step()
        for params, opt, graph in graphs:
            if t == 0:
                continue
            for p, q in zip(params, grads[t]):
                p.grad.copy_(q)
            opt.host_advance()
            graph.replay()
    for params, opt, _ in graphs:
        for p, q in zip(params, eager):
            assert torch.equal(p, q) and all(torch.equal(opt.state[p][n], eo.state[q][n]) for n in eo.state[q])


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 64, 65, 300])
def test_few_and_many_tensors(count):
    """Up to 64 tensors' addresses travel with the launch, those of more lie in a table; either way other tensors of the same sizes are other tensors."""
    sets = []
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        shapes = [(int(torch.randint(1, 700, (1,), generator=g)),) for _ in range(1)] + [(129 + i % 40,) for i in range(count - 1)]
        shapes[0] = (500,)
        s = dict(params=[torch.randn(n, generator=g) for n in shapes], grads=[torch.randn(n, generator=g) for n in shapes])
        s["ms"], s["vs"] = ([torch.zeros(n, dtype=torch.uint8) for n in shapes] for _ in range(2))
        s["mscales"], s["vscales"] = ([torch.zeros(-(-n[0] // 128)) for n in shapes] for _ in range(2))
        s["shadows"] = [None] * count
        sets.append((s, {n: [None if t is None else t.cuda() for t in ts] for n, ts in s.items()}))
    for t in (1, 2):
        for a, b in sets:
            step(a, plain, step=t, seed=t)
            step(b, multi_tensor.adamw8_step, step=t, seed=t)
    for a, b in sets:
        for name in ("ms", "mscales", "vs", "vscales"):
            assert all(torch.equal(x, y.cpu()) for x, y in zip(a[name], b[name])), name
        for signed, codes, scales in ((True, "ms", "mscales"), (False, "vs", "vscales")):
            got = multi_tensor.state8_values(b[codes], b[scales], signed)
            assert all(torch.equal(x.cpu(), oracle.state8_decode(c, sc, signed)) for x, c, sc in zip(got, a[codes], a[scales]))


@pytest.mark.gpu
def test_on_another_stream():
    a, b = problem(6, "cuda"), problem(6, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(a, multi_tensor.adamw8_step, step=2)
    with torch.cuda.stream(side):
        step(b, multi_tensor.adamw8_step, step=2)
        values = multi_tensor.state8_values(b["ms"], b["mscales"], True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for n in ("params", "ms", "vs", "vscales") for x, y in zip(a[n], b[n]))
    assert all(torch.equal(v, w) for v, w in zip(values, multi_tensor.state8_values(a["ms"], a["mscales"], True)))


def test_kernels_off_runs_the_plain_statement():
    ops.force_fallback(True)
    try:
        s = problem(7)
        step(s, multi_tensor.adamw8_step, step=1)
        assert torch.isfinite(s["params"][0]).all()
    finally:
        ops.force_fallback(False)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_a_tensors_number_is_what_its_random_bits_go_by(device):
    """Without numbers: the place in the list.  With them a tensor's step is the same wherever it stands and whatever stands beside it."""
    a, b, c = (problem(11, device) for _ in range(3))
    step(a, multi_tensor.adamw8_step, step=3, seed=4)
    numbers = [7 * i % 10 for i in range(len(SHAPES))]
    step(b, multi_tensor.adamw8_step, step=3, seed=4, numbers=list(range(len(SHAPES))))
    assert all(torch.equal(x, y) for name in a for x, y in zip(a[name], b[name]) if x is not None)
    some = [9, 8, 3, 2]
    c = {name: [ts[i] for i in some] for name, ts in c.items()}
    step(c, multi_tensor.adamw8_step, step=3, seed=4, numbers=some)
    for name in a:
        assert all(x is None or torch.equal(x, y) for x, y in zip((a[name][i] for i in some), c[name])), name
    d, e = problem(11, device), problem(11, "cpu")
    step(d, multi_tensor.adamw8_step, step=3, seed=4, numbers=numbers)
    step(e, plain, step=3, seed=4, numbers=numbers)
    for name in ("ms", "mscales", "vs", "vscales"):
        assert all(torch.equal(x.cpu(), y) for x, y in zip(d[name], e[name])), name
    assert any(not torch.equal(x, y) for x, y in zip(a["ms"], d["ms"]))
    if device == "cuda":
        for bad in (numbers[:-1], [-1] + numbers[1:], [1 << 30] + numbers[1:]):
            with pytest.raises(ValueError):
                step(d, multi_tensor.adamw8_step, step=3, numbers=bad)
        step(d, multi_tensor.adamw8_step, step=3, numbers=[(1 << 30) - 1] + numbers[1:])


@pytest.mark.gpu
def test_numbers_of_many_tensors():
    """More than 64 tensors: addresses from a table; the numbers come with the sizes all the same."""
    g = torch.Generator().manual_seed(1)
    grads = [torch.randn(200 + i, generator=g) for i in range(70)]
    out = []
    for order in (range(70), range(69, -1, -1)):
        s = dict(params=[torch.zeros(200 + i, device="cuda") for i in order], grads=[grads[i].cuda() for i in order], shadows=[None] * 70)
        s["ms"], s["vs"] = ([torch.zeros(200 + i, dtype=torch.uint8, device="cuda") for i in order] for _ in range(2))
        s["mscales"], s["vscales"] = ([torch.zeros(-(-(200 + i) // 128), device="cuda") for i in order] for _ in range(2))
        step(s, multi_tensor.adamw8_step, step=1, seed=2, numbers=[1000 + i for i in order])
        out.append({n: ts if order[0] == 0 else ts[::-1] for n, ts in s.items()})
    assert all(torch.equal(x, y) for n in ("params", "ms", "vs", "mscales", "vscales") for x, y in zip(out[0][n], out[1][n]))


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_a_step_that_leaves_a_parameter_out(device):
    """The others are rounded as they would have been beside it, and a parameter with a number as itself in any group's order."""
    g = torch.Generator().manual_seed(5)
    start, grads = ([torch.randn(n, generator=g) for n in (300, 400, 500)] for _ in range(2))

    def run(order, without=(), numbers=None):
        params = [torch.nn.Parameter(start[i].to(device, copy=True)) for i in order]
        opt = AdamW(params, lr=1e-2, fused=True, state_bits=8)
        if numbers:
            opt.number_tensors({p: numbers[i] for p, i in zip(params, order)})
        for p, i in zip(params, order):
            p.grad = None if i in without else grads[i].to(device, copy=True)
        opt.step()
        return {i: (p.detach(), opt.state[p].get("exp_avg"), opt.state[p].get("exp_avg_sq")) for p, i in zip(params, order)}

    def same(x, y):
        return all(torch.equal(u, v) for u, v in zip(x, y))

    whole, part = run([0, 1, 2]), run([0, 1, 2], without=(0,))
    assert same(whole[1], part[1]) and same(whole[2], part[2])
    numbered, other = run([0, 1, 2], numbers=[4, 9, 17]), run([2, 0], numbers=[4, 9, 17])
    assert same(numbered[2], other[2]) and same(numbered[0], other[0]) and not torch.equal(numbered[2][1], whole[2][1])


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_negative_zeros(device):
    """A first moment that was rounded to -0 and a gradient of -0 (that of nothing, with `maximize`): the code keeps its sign on every device."""
    codes, _ = oracle.state8_encode(torch.tensor([1.0, -0.0, 0.0, -1.0]), torch.zeros(4, dtype=torch.int64), True)
    assert codes.tolist() == [127, 128, 0, 255]
    n = 300
    m = torch.zeros(n)
    m[0], m[128], m[256] = 1.0, 1.0, 1.0
    made, scales = oracle.state8_encode(m, torch.zeros(n, dtype=torch.int64), True)
    made[5:100] = made[200:250] = 128
    s = dict(params=[torch.zeros(n)], grads=[torch.zeros(n)], ms=[made], mscales=[scales], vs=[torch.zeros(n, dtype=torch.uint8)],
             vscales=[torch.zeros(3)], shadows=[None])
    s = {name: [None if t is None else t.to(device) for t in ts] for name, ts in s.items()}
    step(s, multi_tensor.adamw8_step, step=1, maximize=True)
    want = torch.zeros(n, dtype=torch.uint8)
    want[5:100] = want[200:250] = 128
    want[0] = want[128] = want[256] = 127
    assert torch.equal(s["ms"][0].cpu(), want)


def test_what_small_elements_of_a_block_move():
    """400 steps with a constant gradient, eps 0: all elements of a 32-bit step would move alike.  A second moment above zero keeps its first step, 2^-34.9
    of the block's largest, whose root is 2^-17.45: elements down to there move as the largest do, those below are damped in proportion, to
    under a half at the first moment's first step, 2^-18.9.  A mean over 127 elements; single ones scatter by the rounding of both moments."""
    powers = [8, 14, 16, 17, 17.45, 18, 18.9, 20]
    g = torch.stack([torch.full((128,), 2.0 ** -p) for p in powers])
    g[:, 0] = 1.0
    p = torch.zeros_like(g)
    m, v = torch.zeros_like(g, dtype=torch.uint8), torch.zeros_like(g, dtype=torch.uint8)
    ms, vs = torch.zeros(len(powers)), torch.zeros(len(powers))
    for t in range(1, 401):
        oracle.adamw8([p], [g], [m], [ms], [v], [vs], [None], 1e-3, 0.9, 0.95, 0.0, 0.0, t)
    way = -p
    assert torch.allclose(way[:, 0], torch.tensor(0.4), rtol=1e-3)
    moved = dict(zip(powers, way[:, 1:].mean(1).tolist()))
    for power in powers:
        if power <= 17.45:
            assert 0.95 * 0.4 <= moved[power] <= 1.05 * 0.4, (power, moved)      # (an eighth of a code, averaged over steps and elements)
        else:
            floor = 2.0 ** (17.4535 - power)                                     # root of the first step over the element's own
            assert 0.95 * floor * 0.4 <= moved[power] <= 1.1 * floor * 0.4, (power, moved)


def test_how_far_a_first_moment_is_off():
    """One step of its code at most, (|x| + FIRST scale) / 8: an eighth of large values, half of a value at 2^-18, all of one at the first step."""
    for power, most in ((4, 1 / 8), (12, 1 / 8), (15, 1 / 7), (16, 1 / 6), (17, 1 / 4), (18, 1 / 2), (18.9, 1.0)):
        x = torch.full((128,), 2.0 ** -power)
        x[0] = 1.0
        bound = (x[1] + FIRST[True] / TOP[True]) / 8
        for r in range(0, 65536, 257):
            kept = oracle.state8_decode(*oracle.state8_encode(x, torch.full((128,), r), True), True)
            off = float((kept[1] - x[1]).abs())
            assert off <= float(bound) + 2.0 ** -20 * float(x[1]) and off <= most * float(x[1]) * (1 + 2.0 ** -10)
