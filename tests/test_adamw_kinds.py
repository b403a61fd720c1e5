"""AdamW with moments in 8 bits and bf16 parameters: the kernel is the formula bit for bit, and the formula is AdamW's."""
import copy
import math

import pytest
import torch

from mccl_b200.optim import FusedAdamW
from mccl_b200.optim.moments import GROUP, pack_moment, padded, unpack_moment
from mccl_b200.utils.spawn import run_workers

U = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
KINDS = [(torch.float32, 8), (torch.bfloat16, 8), (torch.bfloat16, 32)]


# ---- the formula, one rounding an operation ----------------------------------------------------
def _dither(n, step):
    word = 0xFFFFFFFF
    h = ((torch.arange(n) ^ (step * 0x9E3779B9 & word)) * 0x6A09E667) & word
    h ^= h >> 15
    h = (h * 0xBB67AE85) & word
    h ^= h >> 16
    return h & 0xFFFF, h >> 16


def _codes(x, dither, digits, top):
    """By the real numbers of the format: x between two of its values, and the upper one where the dither reaches it."""
    v = torch.zeros(padded(x.numel()), dtype=torch.float64)
    v[:x.numel()] = x.double()
    r = torch.zeros(v.numel(), dtype=torch.float64)
    r[:x.numel()] = dither.double() / 65536
    v, r = v.view(-1, GROUP), r.view(-1, GROUP)
    most = v.abs().amax(1, keepdim=True)
    # the smallest power of two in whose units the largest is at most 1.75 * 2^top, from 2^-120 on
    mantissa, exponent = torch.frexp(most)
    power = torch.where(most > 0, exponent - 1 - top + (mantissa * 2 > 1.75).int(), -1000).clamp(min=-120)
    y = torch.ldexp(v.abs(), -power)
    some = y.float() > 0
    lowest = -6 if digits == 3 else -14
    # the fp32 formula holds y to 24 digits, and below the lowest binade to as many as there are beside 2^lowest
    y = torch.where(y < 2.0 ** lowest, (y + 2.0 ** lowest).float().double() - 2.0 ** lowest, y)
    step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=lowest).double() - digits)
    below = torch.floor(y / step)
    units = below + ((y / step - below) + r >= 1).double()
    value = units * step
    if digits == 2:
        value = torch.where(some, value.clamp(min=2.0 ** (lowest - digits)), value)
    value = torch.copysign(value, v)
    bad = ~torch.isfinite(most)
    return torch.where(bad, 0.0, value).view(-1), torch.where(bad, math.nan, torch.ldexp(torch.ones_like(most), power)).view(-1).float()


class Formula:
    """One tensor's step on the CPU."""

    def __init__(self, p, bits):
        self.half, self.bits, self.n, self.shape = p.dtype is torch.bfloat16, bits, p.numel(), p.shape
        self.p = p.detach().cpu().float().reshape(-1)
        self.m = [torch.zeros(padded(self.n)).double(), torch.zeros(padded(self.n) // GROUP)] if bits == 8 else [torch.zeros(self.n)]
        self.v = [t.clone() for t in self.m]
        self.t = 0

    @staticmethod
    def _value(state, n):
        if len(state) == 1:
            return state[0]
        return (state[0].float().view(-1, GROUP) * state[1][:, None]).view(-1)[:n]

    def step(self, grad, lr, betas, eps, weight_decay):
        self.t += 1
        (b1, b2), g = betas, grad.detach().cpu().float().reshape(-1)
        m, v = self._value(self.m, self.n), self._value(self.v, self.n)
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * (1 - b2) * g
        root = torch.sqrt(v.double()).float()  # correctly rounded, which a root in 32 bits need not be on every CPU
        below = root * (1 / math.sqrt(1 - b2 ** self.t)) + eps
        self.p = self.p * (1 - lr * weight_decay) - m / below * (lr / (1 - b1 ** self.t))
        if self.bits == 8:
            lower, upper = _dither(self.n, self.t)
            self.m, self.v = list(_codes(m, lower, 3, 8)), list(_codes(v, upper, 2, 15))
        else:
            self.m, self.v = [m], [v]

    def check(self, p, state):
        where = f"step {self.t}, {self.n} numbers"
        if self.half:
            whole = (p.detach().cpu().reshape(-1).view(torch.int16).int() << 16) + state["low"].cpu().reshape(-1).int()
            assert torch.equal(whole.view(torch.float32), self.p), where
        else:
            assert torch.equal(p.detach().cpu().reshape(-1), self.p), where
        for name, own in (("exp_avg", self.m), ("exp_avg_sq", self.v)):
            assert torch.equal(state[name].cpu().float().reshape(-1), own[0].float()), (where, name)
            if self.bits == 8:
                assert torch.equal(state[name + "_scale"].cpu(), own[1]), (where, name)


# ---- without a GPU -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind,step", [(torch.float8_e4m3fn, 2.0 ** -3), (torch.float8_e5m2, 2.0 ** -2)])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 1000])
def test_packed_moments_are_half_a_step_away(kind, step, n):
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen))
    if kind is torch.float8_e5m2:
        x = x.square()
    codes, scale = pack_moment(x, kind)
    assert codes.dtype is kind and codes.numel() == padded(n) and scale.numel() == padded(n) // GROUP and torch.isfinite(codes.float()).all()
    back = unpack_moment(codes, scale, x.shape)
    least = scale.repeat_interleave(GROUP)[:n] * 2.0 ** (-9 if kind is torch.float8_e4m3fn else -16)
    # half a step of at most `step` of the value, or below the lowest binade half of its step, where a square also stays above zero
    assert ((back - x).abs() <= x.abs() * step / 2 + least).all()
    again = pack_moment(back, kind)
    assert torch.equal(unpack_moment(*again, x.shape), back)


def test_a_group_that_is_not_finite_is_nan():
    x = torch.ones(600)
    x[300] = math.inf
    back = unpack_moment(*pack_moment(x, torch.float8_e4m3fn), x.shape)
    assert torch.isnan(back[256:512]).all() and torch.equal(back[:256], x[:256]) and torch.equal(back[512:], x[512:])
    assert pack_moment(torch.zeros(0), torch.float8_e5m2)[0].numel() == 0


def test_refusals_without_a_gpu():
    p = [torch.nn.Parameter(torch.ones(4))]
    with pytest.raises(ValueError, match="state_bits"):
        FusedAdamW(p, state_bits=16)
    opt = FusedAdamW(p, state_bits=8)
    p[0].grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="float32 or bfloat16 CUDA"):
        opt.step()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("into", [8, 32])
def test_checkpoints_of_either_kind_load_into_the_other(dtype, bits, into):
    torch.manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(*s).to(dtype)) for s in ((30, 20), (5,))]
    a, b = FusedAdamW(params, state_bits=bits), FusedAdamW(params, state_bits=into)
    for p in params:
        st = a._state_of(p)
        st["step"] = torch.tensor(7.0)
        for name, kind in (("exp_avg", torch.float8_e4m3fn), ("exp_avg_sq", torch.float8_e5m2)):
            x = torch.rand(p.shape) + 1e-3
            if bits == 8:
                st[name], st[name + "_scale"] = pack_moment(x, kind)
            else:
                st[name] = x
        if dtype is torch.bfloat16:
            st["low"] = torch.randint(-32768, 32768, p.shape, dtype=torch.int16)
    kept = copy.deepcopy(a.state_dict())
    b.load_state_dict(kept)
    for p in params:
        assert float(b.state[p]["step"]) == 7
        assert ("exp_avg_scale" in b.state[p]) == (into == 8)
        assert b.state[p]["exp_avg"].dtype is (torch.float8_e4m3fn if into == 8 else torch.float32)
        if dtype is torch.bfloat16:
            assert torch.equal(b.state[p]["low"], a.state[p]["low"])
        for x, y, step in zip(a.moments(p), b.moments(p), (2.0 ** -4, 2.0 ** -3)):
            # the same where nothing is rounded (what was packed before is a value of the format), else half a step
            assert torch.equal(x, y) if bits == 8 or into == 32 else ((x - y).abs() <= x * step).all()
    mine = torch.optim.AdamW(params)
    for p in params:
        p.grad = torch.full_like(p, 0.5)
    mine.step()
    b.load_state_dict(mine.state_dict())
    for p in params:
        x = mine.state[p]["exp_avg"].float()
        assert ((b.moments(p)[0] - x).abs() <= x.abs() * 2.0 ** -4).all() and b.moments(p)[0].dtype is torch.float32


# ---- the kernel ---------------------------------------------------------------------------------
SIZES = [(1,), (7,), (255,), (256,), (257,), (3, 1000), (4096,), (4097,), (70001,)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_steps_are_the_formula_bit_for_bit(cuda_device, dtype, bits):
    torch.manual_seed(11)
    params = [torch.nn.Parameter(torch.randn(s, device=cuda_device).to(dtype)) for s in SIZES]
    own = [Formula(p, bits) for p in params]
    opt = FusedAdamW(params, state_bits=bits, **HYPER)
    for i in range(6):
        for p, f in zip(params, own):
            # numbers of every size, zeros among them; whole tensors of zeros and of tiny numbers
            g = torch.randn_like(p) * torch.exp(4 * torch.randn_like(p)) * (torch.rand_like(p) < 0.8)
            p.grad = (g * (0.0 if i == 2 else 1e-18 if i == 3 else 1.0)).to(dtype)
            f.step(p.grad, **HYPER)
        opt.step()
        for p, f in zip(params, own):
            f.check(p, opt.state[p])


@pytest.mark.gpu
def test_roots_and_quotients_are_correctly_rounded(cuda_device):
    import mccl_b200
    native = mccl_b200.require_native()
    # every number of two neighbouring binades: a root's digits depend on no more, and a reciprocal's on one of them
    b = torch.arange(1 << 24, dtype=torch.int32, device=cuda_device).add_(0x3F800000).view(torch.float32)
    root, quotient = native._test_root_quotient(torch.ones_like(b), b)
    assert torch.equal(root, torch.sqrt(b.double()).float()) and torch.equal(quotient, torch.ones_like(b) / b)
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    for near in (False, True):  # numerators of every kind, and ones beside a multiple of the denominator
        for scale in (2.0 ** -58, 2.0 ** -31, 1.0, 2.0 ** 25):
            a = torch.randn(b.shape, generator=gen, device=cuda_device) * scale
            a = b * (torch.randint(1, 1 << 24, b.shape, generator=gen, device=cuda_device).float() * 2.0 ** -23) * scale if near else a
            inside = (a.abs() >= 2.0 ** -60) & (a.abs() <= 2.0 ** 60)
            assert torch.equal(torch.where(inside, native._test_root_quotient(a, b)[1], 0), torch.where(inside, a / b, 0))
    small = b * 2.0 ** -60
    assert torch.equal(native._test_root_quotient(b, small)[0], torch.sqrt(small.double()).float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_tensors_that_are_not_aligned(cuda_device, dtype, bits):
    torch.manual_seed(12)
    storage, grads = (torch.randn(5000, device=cuda_device).to(dtype) for _ in range(2))
    around = storage.clone()
    params = [torch.nn.Parameter(storage[1:2001]), torch.nn.Parameter(storage[2002:4002])]
    own = [Formula(p, bits) for p in params]
    opt = FusedAdamW(params, state_bits=bits, **HYPER)
    for i in range(3):
        for p, f, at in zip(params, own, (0, 2003)):
            p.grad = grads[at + i:at + i + 2000]
            f.step(p.grad, **HYPER)
        opt.step()
        for p, f in zip(params, own):
            f.check(p, opt.state[p])
    for at in (slice(0, 1), slice(2001, 2002), slice(4002, 5000)):
        assert torch.equal(storage[at], around[at])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_a_step_is_adamw_in_64_bits(cuda_device, dtype, bits):
    torch.manual_seed(13)
    p = torch.nn.Parameter(torch.randn(5000, device=cuda_device).to(dtype))
    opt = FusedAdamW([p], state_bits=bits, **HYPER)
    (b1, b2), lr, wd = HYPER["betas"], HYPER["lr"], HYPER["weight_decay"]
    for t in range(1, 4):
        low = opt.state[p]["low"].int() if t > 1 and dtype is torch.bfloat16 else 0
        before = p.detach().float().double() if dtype is torch.float32 else ((p.detach().view(torch.int16).int() << 16) + low).view(torch.float32).double()
        m, v = (x.double() for x in opt.moments(p))
        g = torch.randn_like(p)
        p.grad = g
        opt.step()
        m, v = b1 * m + (1 - b1) * g.double(), b2 * v + (1 - b2) * g.double() ** 2
        move = lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"])
        want = before * (1 - lr * wd) - move
        # m: three roundings of its terms' sizes; v: four, halved by the root; root, product, sum, quotient, product and the constants: 12
        # of the move's largest term.  p: the product's and the difference's, and of bf16 the half step of what is returned.
        terms = lr * ((m.abs() + 2 * (1 - b1) * g.double().abs()) / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"])
        bound = 2 * U * before.abs() + 15 * U * terms + (2.0 ** -8 * want.abs() if dtype is torch.bfloat16 else 0)
        assert ((p.detach().double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_small_changes_of_the_second_moment_add_up(cuda_device):
    n, steps = 1 << 16, 300
    p = torch.nn.Parameter(torch.zeros(n, device=cuda_device))
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    size = torch.exp(torch.randn(n, generator=gen, device=cuda_device))
    opt = FusedAdamW([p], lr=1e-3, state_bits=8)
    for _ in range(steps):
        p.grad = size
        opt.step()
    share = opt.moments(p)[1].double() / (size.double() ** 2 * (1 - 0.999 ** steps))
    # Every step adds a thousandth of g^2 and moves v, by chance, by a step of at most a quarter of v: the variance of one move is at most the
    # move times the step, 0.00025 g^2 v, and that of their sum below 300 of them, 0.075 of g^4 at most 0.26 g^2 each: 0.02 g^4, 0.28 of the
    # share's 0.26^2.  Of 65536 numbers the mean is within 0.53 / 256; six of these.  (Rounded to nearest v would stop at 0.008 g^2, a share of 0.03.)
    assert abs(float(share.mean()) - 1) < 6 * 0.53 / 256
    assert float(share.var()) < 0.28 * 1.1
    # m settles within steps, 0.1 g + 0.9 m by chance up or down by an eighth: variance of a move 1/4 of a step squared, summed over 0.81^k
    first = opt.moments(p)[0].double() / size.double()
    assert abs(float(first.mean()) - 1) < 6 * math.sqrt(1 / 64 / 4 / (1 - 0.81)) / 256


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_an_infinite_gradient_stays_in_its_group(cuda_device, dtype, bits):
    p = torch.nn.Parameter(torch.ones(1000, device=cuda_device, dtype=dtype))
    opt = FusedAdamW([p], state_bits=bits, **HYPER)
    g = torch.ones_like(p)
    g[300] = math.inf
    for _ in range(2):
        p.grad = g
        opt.step()
    bad = torch.zeros(1000, dtype=torch.bool, device=cuda_device)
    bad[slice(256, 512) if bits == 8 else slice(300, 301)] = True
    assert torch.equal(torch.isnan(p.detach()), bad)
    if dtype is torch.bfloat16:
        assert torch.isfinite(p.detach()[~bad]).all()


@pytest.mark.gpu
def test_a_bf16_parameter_that_the_program_changes(cuda_device):
    p = torch.nn.Parameter(torch.randn(512, device=cuda_device).bfloat16())
    opt = FusedAdamW([p], state_bits=8, lr=1e-5, weight_decay=0.0)
    for _ in range(3):
        p.grad = torch.randn_like(p)
        opt.step()
    with torch.no_grad():
        p[:256].zero_()
        p[256:].fill_(3.0)
    p.grad = torch.zeros_like(p)
    opt.step()
    assert torch.isfinite(p.detach()).all()
    # a step is at most lr / 0.1 * 1.1 or so of what was left of m; what was below the parameter, half a step of bf16
    assert (p.detach()[:256].float().abs() < 2e-3).all() and ((p.detach()[256:].float() - 3).abs() <= 2 ** -6).all()


@pytest.mark.gpu
def test_small_steps_of_a_bf16_parameter_add_up(cuda_device):
    start = torch.full((300,), 2.0, device=cuda_device)
    p, q = torch.nn.Parameter(start.bfloat16()), torch.nn.Parameter(start.clone())
    a, b = FusedAdamW([p], state_bits=8, lr=1e-4, weight_decay=0.0), FusedAdamW([q], state_bits=8, lr=1e-4, weight_decay=0.0)
    for _ in range(200):  # each an 80th of a step of bf16
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
        a.step(), b.step()
    assert torch.equal(p.detach(), q.detach().bfloat16()) or (p.detach().float() - q.detach()).abs().max() <= 2.0 ** -8 * 2
    assert (p.detach() < 2.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_a_resumed_run_is_the_uninterrupted_one(cuda_device, dtype, bits):
    torch.manual_seed(14)
    params = [torch.nn.Parameter(torch.randn(s, device=cuda_device).to(dtype)) for s in ((700,), (33, 7))]
    opt = FusedAdamW(params, state_bits=bits, **HYPER)
    grads = [[torch.randn_like(p) for p in params] for _ in range(6)]

    def run(params, opt, some):
        for gs in some:
            for p, g in zip(params, gs):
                p.grad = g.clone()
            opt.step()

    run(params, opt, grads[:3])
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = FusedAdamW(copies, state_bits=bits, **HYPER)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    run(params, opt, grads[3:])
    run(copies, other, grads[3:])
    for p, q in zip(params, copies):
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.moments(p), other.moments(q)))


@pytest.mark.gpu
def test_kinds_side_by_side_in_one_launch_and_on_another_stream(cuda_device):
    import mccl_b200
    native = mccl_b200.require_native()
    torch.manual_seed(15)
    params = [torch.nn.Parameter(torch.randn(999, device=cuda_device).to(d)) for d in (torch.bfloat16, torch.float32, torch.bfloat16)]
    params.append(torch.nn.Parameter(torch.randn(50, device=cuda_device)))
    params[3].requires_grad_(False)
    own = [Formula(p, 32) for p in params[:3]]
    opt = FusedAdamW(params[:3], **HYPER)
    side = torch.cuda.Stream()
    for _ in range(3):
        for p, f in zip(params, own):
            p.grad = torch.randn_like(p)
            f.step(p.grad, **HYPER)
        side.wait_stream(torch.cuda.current_stream())
        before = native._kernel_launches()
        with torch.cuda.stream(side):
            opt.step()
        assert native._kernel_launches() == before + 1
        torch.cuda.current_stream().wait_stream(side)
        for p, f in zip(params, own):
            f.check(p, opt.state[p])


@pytest.mark.gpu
def test_refusals(cuda_device):
    import mccl_b200
    native = mccl_b200.require_native()
    p = torch.nn.Parameter(torch.ones(8, device=cuda_device, dtype=torch.float16))
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        FusedAdamW([p]).step()
    q = torch.ones(300, device=cuda_device)
    m, v = torch.zeros(512, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn), torch.zeros(512, dtype=torch.uint8, device=cuda_device).view(torch.float8_e5m2)
    s = torch.zeros(2, device=cuda_device)
    native.AdamWPlan([q], [m], [v], [(s, s.clone(), None)])
    for params, ms, vs, extra in (([q], [m], [m], (s, s, None)), ([q], [m[:300]], [v], (s, s, None)), ([q], [m], [v], (s, s[:1], None)),
                                  ([q], [m], [v], (s, None, None)), ([q], [m], [v], (s, s, torch.zeros(300, dtype=torch.int16, device=cuda_device))),
                                  ([q.bfloat16()], [m], [v], (s, s, None)), ([q.half()], [m], [v], (s, s, None)), ([q], [q.cpu()], [q], (None, None, None))):
        with pytest.raises(RuntimeError, match="AdamWPlan"):
            native.AdamWPlan(params, ms, vs, [extra])
    plan = native.AdamWPlan([q], [m], [v], [(s, s.clone(), None)])
    with pytest.raises(RuntimeError, match="gradient 0"):
        plan.step([q.bfloat16()], 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_a_captured_step_is_refused_and_does_nothing(cuda_device, dtype, bits):
    p = torch.nn.Parameter(torch.randn(1000, device=cuda_device).to(dtype))
    opt = FusedAdamW([p], state_bits=bits)
    p.grad = torch.randn_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.synchronize()
    before = [p.detach().clone(), *opt.moments(p)]
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            opt.step()
    torch.cuda.synchronize()
    assert float(opt.state[p]["step"]) == 1 and all(torch.equal(a, b) for a, b in zip(before, [p.detach(), *opt.moments(p)]))
    opt.step()
    assert float(opt.state[p]["step"]) == 2 and not torch.equal(before[0], p.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_what_a_block_takes_does_not_show(cuda_device, dtype, bits):
    # 24 Mi numbers and more in all go by larger parts than fewer do
    sizes = [1, 255, 8191, 8193, 20000, 100000]
    sizes.append((24 << 20) - sum(sizes))
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    values = [torch.randn(n, device=cuda_device, generator=gen).to(dtype) for n in sizes]
    grads = [torch.randn(n, device=cuda_device, generator=gen).to(dtype) for n in sizes]

    def steps(which):
        params = [torch.nn.Parameter(values[i].clone()) for i in which]
        opt = FusedAdamW(params, lr=1e-2, state_bits=bits)
        for _ in range(3):
            for p, i in zip(params, which):
                p.grad = grads[i]
            opt.step()
        return [(p.detach(), opt.state[p]) for p in params]

    together, apart = steps(range(7)), steps(range(6)) + steps([6])
    for (p, s), (q, t) in zip(together, apart):
        assert torch.equal(p, q)
        for k in s:
            assert torch.equal(s[k].view(torch.uint8) if s[k].element_size() == 1 else s[k], t[k].view(torch.uint8) if t[k].element_size() == 1 else t[k]), k


def _in_backward(rank, ws):
    import os
    import torch
    from mccl_b200.optim import FusedAdamW
    from mccl_b200.parallel import wrap_ddp

    dtype, bits = getattr(torch, os.environ["TEST_DTYPE"]), int(os.environ["TEST_BITS"])

    def make():
        torch.manual_seed(3)
        return torch.nn.Sequential(torch.nn.Linear(128, 512), torch.nn.GELU(), torch.nn.Linear(512, 8)).to(device, dtype)

    a, b = make(), make()
    oa, ob = (FusedAdamW(m.parameters(), lr=1e-3, state_bits=bits) for m in (a, b))
    da = wrap_ddp(a, device_ids=[device.index], bucket_cap_mb=1)
    db = wrap_ddp(b, device_ids=[device.index], bucket_cap_mb=1, optimizer_in_backward=ob)
    for i in range(4):
        x, y = torch.randn(8, 128, device=device).to(dtype), torch.randint(0, 8, (8,), device=device)
        for d, o in ((da, oa), (db, ob)):
            o.zero_grad()
            torch.nn.functional.cross_entropy(d(x).float(), y).backward()
            o.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and all(torch.equal(x, y) for x, y in zip(oa.moments(p), ob.moments(q)))
        assert float(ob.state[q]["step"]) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("python_hook", ["0", "1"])
@pytest.mark.parametrize("dtype,bits", [("float32", 8), ("bfloat16", 8), ("bfloat16", 32)])
def test_updated_inside_backward(python_hook, dtype, bits):
    env = {"MCCL_PYTHON_BUCKET_HOOK": python_hook, "TEST_DTYPE": dtype, "TEST_BITS": str(bits)}
    run_workers(_in_backward, 1, device="cuda", timeout=180, env=env)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [("exp_avg_scale",), ("exp_avg_sq_scale",), ("exp_avg_scale", "exp_avg_sq_scale")])
def test_moments_of_32_bits_beside_scales_are_refused(cuda_device, dtype, which):
    p = torch.nn.Parameter(torch.ones(300, device=cuda_device, dtype=dtype))
    opt = FusedAdamW([p])
    for name in which:
        opt._state_of(p)[name] = torch.ones(2, device=cuda_device)
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="without scales"):
        opt.step()
    assert torch.equal(p, torch.ones_like(p)) and float(opt.state[p]["step"]) == 0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype,other", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("into", [8, 32])
def test_checkpoints_load_into_parameters_of_another_type(device, dtype, other, bits, into):
    gen = torch.Generator().manual_seed(5)
    first = [torch.randn(*s, generator=gen).to(device, dtype).requires_grad_() for s in ((30, 20), (5,))]
    a = FusedAdamW(first, state_bits=bits, **HYPER)
    for p in first:
        st = a._state_of(p)
        st["step"] = torch.tensor(7.0)
        for name, kind in (("exp_avg", torch.float8_e4m3fn), ("exp_avg_sq", torch.float8_e5m2)):
            x = (torch.rand(p.shape, generator=gen) + 1e-3).to(device)
            if bits == 8:
                st[name], st[name + "_scale"] = pack_moment(x, kind)
            else:
                st[name] = x
        if dtype is torch.bfloat16:
            st["low"] = torch.randint(-32768, 32768, p.shape, generator=gen, dtype=torch.int16).to(device)
    second = [p.detach().to(other, copy=True).requires_grad_() for p in first]
    b = FusedAdamW(second, state_bits=into, **HYPER)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    names = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if into == 8 else set())
    for p, q in zip(first, second):
        st = b.state[q]
        assert set(st) - {"low"} == names and ("low" in st) == (dtype is other is torch.bfloat16) and float(st["step"]) == 7
        if "low" in st:
            assert torch.equal(st["low"], a.state[p]["low"])
        for x, y, step in zip(a.moments(p), b.moments(q), (2.0 ** -4, 2.0 ** -3)):
            assert torch.equal(x, y) if bits == 8 or into == 32 else ((x - y).abs() <= x * step).all()
    if device == "cpu":
        return
    for q in second:
        q.grad = torch.ones_like(q)
    b.step()
    for p, q in zip(first, second):
        # (the step, 3e-4, is less than a bf16 number of size one shows)
        moved = not torch.equal(q, p.detach().to(other)) or (other is torch.bfloat16 and not torch.equal(b.state[q]["low"], a.state[p].get("low", torch.zeros_like(b.state[q]["low"]))))
        assert float(b.state[q]["step"]) == 8 and torch.isfinite(q).all() and moved
        # m = 0.9 m + 0.1 of what was loaded, itself half a step off where it was packed; a step of 8 bits is an eighth at most
        want = a.moments(p)[0] * 0.9 + 0.1
        loaded = 0.0 if bits == 8 or into == 32 else 2.0 ** -4
        assert ((b.moments(q)[0] - want).abs() <= want * (loaded + (2.0 ** -3 * (1 + loaded) if into == 8 else 0.0) + 2.0 ** -20)).all()


@pytest.mark.gpu
def test_quotients_beside_the_middle_of_two_numbers(cuda_device):
    import mccl_b200
    native = mccl_b200.require_native()
    hard = [(float.fromhex(a), float.fromhex(b)) for a, b in (("0x1.aaaaa6p0", "0x1.fffffap0"), ("0x1p0", "0x1.fffffep0"), ("0x1.fffffcp0", "0x1.fffffep0"))]
    a, b = (torch.tensor(v, device=cuda_device) for v in zip(*hard))
    assert torch.equal(native._test_root_quotient(a, b)[1], (a.double() / b.double()).float())
    # a = A and b = 2^j B with B odd, both of 24 digits: a / b is r / (2 B) units beside Q + 1/2 where (2 Q + 1) B = A 2^k + r, which fixes Q by B's
    # inverse modulo 2^k.  (A quotient of such numbers rounded to 64 bits first is rounded alike.)
    for j in range(5):
        odd = torch.arange((1 << (23 - j)) + 1, 1 << (24 - j), 2, device=cuda_device)
        for k in (24 - j, 25 - j):
            inverse = odd.clone()
            for _ in range(5):
                inverse = (inverse * (2 - odd * inverse)) & ((1 << k) - 1)
            for r in range(1 - (32 >> j), 32 >> j, 2):  # all within 2^-20
                for more in range((1 << 25) >> k):
                    middle = ((inverse * r) & ((1 << k) - 1)) + (more << k)
                    numerator = (middle * odd - r) >> k
                    assert bool(((middle * odd - r) == numerator << k).all())
                    inside = (middle >= 1 << 24) & (numerator >= 1 << 23) & (numerator < 1 << 24)
                    a, b = numerator[inside].float(), odd[inside].float()
                    assert torch.equal(native._test_root_quotient(a, b)[1], (a.double() / b.double()).float())
