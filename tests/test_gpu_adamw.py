"""``addernetcuda_amd.optim.AdamW`` against the rule in 64 bits, and against ``torch.optim.AdamW`` where their states are alike.

Bounds: a moment is a sum of two rounded products (4 u of their sizes), the parameter one rounding of its own and a few of its
update; an 8-bit code is the nearest in its root's scale up to what the roots' own roundings (1e-3 of a code at most) can move."""
import copy

import pytest
import torch

from tests.layer_bounds import U, V

pytestmark = pytest.mark.gpu
SHAPES = [(16, 3, 3, 3), (16,), (64, 64, 3, 3), (10, 64), (5, 7), (1,), (255,), (256,), (257,), (1023,), (1025,), (4095,), (4096,), (4097,),
          (70, 130), (300, 301)]
BLOCK = 256


def params(dtype, seed, shapes=SHAPES):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in shapes]


def set_grads(ps, seed):
    g = torch.Generator().manual_seed(seed)
    for p in ps:
        scale = torch.exp(2 * torch.randn(p.shape, generator=g)) * 1e-2
        p.grad = (torch.randn(p.shape, generator=g) * scale).to(p.dtype).cuda()


def decode(state, name):
    """A moment as float64 on the CPU, by the documented rule."""
    m = state[name].detach().cpu()
    if m.dtype == torch.float32:
        return m.double()
    s = state[name + "_scale"].cpu().double().repeat_interleave(BLOCK)[: m.numel()].view(m.shape)
    q = m.double()
    return s * q * q.abs() / 127 ** 2 if m.dtype == torch.int8 else s * (q / 255) ** 4


def check_moment(state, name, want, off):
    got = state[name].detach().cpu()
    if got.dtype == torch.float32:
        far = (got.double() - want).abs()
        assert (far <= off).all(), (name, far.max())
        return
    n = want.numel()
    w = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64)
    w[:n] = want.flatten()
    w = w.view(-1, BLOCK)
    s = w.abs().amax(1)
    assert torch.allclose(state[name + "_scale"].cpu().double(), s, rtol=8 * U, atol=0), name
    q = got.double().flatten()
    root = (w.abs() / s.clamp(min=1e-300)[:, None]).flatten()[:n]
    if got.dtype == torch.int8:
        assert (q * want.flatten() >= 0).all()
        assert ((127 * root.sqrt() - q.abs()).abs() <= 0.501).all()
    else:
        assert ((255 * root ** 0.25 - q).abs()[q > 1] <= 0.501).all()
        assert ((q > 0) == (want.flatten() > 0)).all() and (255 * root[q <= 1] ** 0.25 <= 1.501).all()


def step_and_check(opt, ps, seed, t, lr, betas, eps, wd):
    set_grads(ps, seed)
    before = []
    for p in ps:
        state = opt.state.get(p)
        zero = torch.zeros(p.shape, dtype=torch.float64)
        before.append((p.detach().double().cpu(), decode(state, "exp_avg") if state else zero, decode(state, "exp_avg_sq") if state else zero))
    opt.step()
    b1, b2 = betas
    for p, (p0, m0, v0) in zip(ps, before):
        g = p.grad.double().cpu()
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        update = lr / (1 - b1 ** t) * m / (v.sqrt() / (1 - b2 ** t) ** 0.5 + eps)
        want = p0 * (1 - lr * wd) - update
        # (the moments' roundings reach the update as they stand to the moments themselves)
        off_m = 6 * U * ((b1 * m0).abs() + ((1 - b1) * g).abs())
        off = 3 * U * p0.abs() + 16 * U * update.abs() + off_m / m.abs().clamp(min=1e-300) * update.abs()
        if p.dtype == torch.bfloat16:
            off = off + V * want.abs()
        far = (p.detach().double().cpu() - want).abs()
        assert (far <= off + 1e-30).all(), (tuple(p.shape), far.max(), off[far > off])
        check_moment(opt.state[p], "exp_avg", m, off_m + 1e-45)
        check_moment(opt.state[p], "exp_avg_sq", v, 8 * U * v + 1e-45)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_steps(dtype, bits, capturable, gpu):
    from addernetcuda_amd.optim import AdamW
    ps = params(dtype, 1)
    rule = dict(lr=1e-2, betas=(0.9, 0.98), eps=1e-8)
    lr = torch.tensor(1e-2, device="cuda") if capturable else 1e-2
    opt = AdamW(ps, lr=lr, betas=rule["betas"], eps=1e-8, weight_decay=0.05, state_bits=bits, capturable=capturable, min_8bit_size=257)
    rule["lr"] = float(lr)
    for t in (1, 2, 3):
        step_and_check(opt, ps, 50 + t, t, wd=0.05, **rule)
    coded = [p for p in ps if opt.state[p]["exp_avg"].dtype == torch.int8]
    assert len(coded) == (sum(p.numel() >= 257 for p in ps) if bits == 8 else 0)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_odd_addresses_and_late_starters(bits, gpu):
    """More tensors than one launch takes, at addresses off any alignment; parameters whose first gradient comes later count for
    themselves."""
    from addernetcuda_amd.optim import AdamW
    base = torch.randn(200 * 700 + 3, device="cuda")
    ps = [torch.nn.Parameter(base[1 + 700 * i: 1 + 700 * i + 650 + i % 40]) for i in range(200)]
    opt = AdamW(ps, lr=1e-2, weight_decay=0.0, state_bits=bits, min_8bit_size=300)
    rule = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, wd=0.0)
    step_and_check(opt, ps, 3, 1, **rule)
    late = torch.nn.Parameter(torch.randn(500, device="cuda"))
    opt.add_param_group({"params": [late]})
    opt.param_groups[0]["params"].append(opt.param_groups.pop()["params"][0])
    set_grads(ps + [late], 4)
    ps[0].grad = None
    opt.step()
    assert opt.state[late]["step"] == 1 and opt.state[ps[1]]["step"] == 2 and opt.state[ps[0]]["step"] == 1
    step_and_check(opt, ps[1:], 5, 3, **rule)


@pytest.mark.parametrize("amsgrad", [False, True])
def test_state_moves_to_and_from_torch(amsgrad, gpu):
    from addernetcuda_amd.optim import AdamW
    ours, ref = params(torch.float32, 2), params(torch.float32, 2)
    kw = dict(lr=3e-3, betas=(0.9, 0.99), weight_decay=0.02, amsgrad=amsgrad)
    o, r = AdamW(ours, **kw), torch.optim.AdamW(ref, **kw)
    for t in range(3):
        set_grads(ours, t)
        set_grads(ref, t)
        o.step()
        r.step()
    for a, b in zip(ours, ref):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)
    r2 = torch.optim.AdamW(ours, **kw)
    r2.load_state_dict(o.state_dict())
    o2 = AdamW(ref, **kw)
    o2.load_state_dict(r.state_dict())
    for t in range(3, 5):
        set_grads(ours, t)
        set_grads(ref, t)
        r2.step()
        o2.step()
    for a, b in zip(ours, ref):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_dict_keeps_every_bit(bits, dtype, capturable, gpu):
    from addernetcuda_amd.optim import AdamW
    a = params(dtype, 6)
    kw = dict(lr=1e-2, state_bits=bits, capturable=capturable)
    oa = AdamW(a, **kw)
    for t in range(2):
        set_grads(a, t)
        oa.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = AdamW(b, **kw)
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    for ps, o in ((a, oa), (b, ob)):
        set_grads(ps, 9)
        o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for name, value in oa.state[p].items():
            other = ob.state[q][name]
            assert torch.equal(value, other) if isinstance(value, torch.Tensor) else value == other
            assert not isinstance(value, torch.Tensor) or (value.dtype == other.dtype and value.data_ptr() != other.data_ptr())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits, gpu):
    from addernetcuda_amd.optim import AdamW
    lr = torch.tensor(1e-2, device="cuda")
    a, b = params(torch.float32, 8), params(torch.float32, 8)
    oa, ob = (AdamW(ps, lr=lr, state_bits=bits, capturable=True, min_8bit_size=257) for ps in (a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        set_grads(a, 0)
        oa.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            oa.step()
    torch.cuda.current_stream().wait_stream(side)
    set_grads(b, 0)
    ob.step()
    grads = [p.grad for p in a]
    for t in range(1, 5):
        lr.fill_(1e-2 / t)
        set_grads(b, t)
        for mine, p in zip(grads, b):
            mine.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        ob.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q), t
            assert torch.equal(oa.state[p]["exp_avg"], ob.state[q]["exp_avg"])
    assert float(oa.state[a[0]]["step"]) == 5


def test_groups_that_the_kernel_leaves(gpu):
    """Parameters that are not contiguous go to torch, beside a group that does not; their state carries over when they come back."""
    from addernetcuda_amd.optim import AdamW
    a = params(torch.float32, 3, [(40, 50), (30, 20)])
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    kw = dict(lr=1e-2, weight_decay=0.1)
    o, r = AdamW([{"params": a[:1]}, {"params": a[1:]}], **kw), torch.optim.AdamW(b, **kw)
    for t in range(4):
        set_grads(a, t)
        set_grads(b, t)
        if t in (1, 2):
            a[1].grad = a[1].grad.t().contiguous().t()
        o.step()
        r.step()
        for p, q in zip(a, b):
            assert torch.allclose(p, q, rtol=1e-6, atol=1e-6), t


@pytest.mark.parametrize("name,codes", [("first", torch.int8), ("second", torch.uint8)])
@pytest.mark.parametrize("n", [1, 255, 256, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_state_values(name, codes, n, dtype, gpu):
    from addernetcuda_amd.optim import state_values
    low, high = (-127, 128) if codes == torch.int8 else (0, 256)
    q = torch.randint(low, high, (n,), dtype=torch.int16).to(codes).cuda()
    s = torch.rand(-(-n // BLOCK), device="cuda")
    got = state_values(q, s, dtype)
    x = q.double() / (high - 1)
    want = s.double().repeat_interleave(BLOCK)[:n] * (x * x.abs() if codes == torch.int8 else x ** 4)
    assert got.dtype == dtype and torch.allclose(got.double(), want, rtol=(6 * U + (V if dtype == torch.bfloat16 else 0)), atol=0)


def test_zero_tiny_and_broken_gradients_in_8_bits(gpu):
    """Blocks of zeros stay zero and do not divide by it; gradients whose squares vanish still move nothing to infinity; an infinite
    gradient spoils its own block (and no other), as the documentation says."""
    from addernetcuda_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(4 * BLOCK + 5, device="cuda"))
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8, min_8bit_size=1)
    g = torch.zeros_like(p)
    g[BLOCK:2 * BLOCK] = 1e-30
    g[2 * BLOCK + 3] = float("inf")
    g[3 * BLOCK:4 * BLOCK] = torch.logspace(-18, 0, BLOCK)
    p.grad = g
    for _ in range(2):
        opt.step()
    state = opt.state[p]
    assert torch.equal(p[:BLOCK], torch.ones(BLOCK, device="cuda")) and not state["exp_avg"][:BLOCK].any()
    assert torch.isfinite(p[:2 * BLOCK]).all() and torch.isfinite(p[3 * BLOCK:]).all()
    assert torch.isnan(state["exp_avg_scale"][2]) and torch.isnan(p[2 * BLOCK:3 * BLOCK]).all()
    # Where the codes run out a first moment may be rounded up to 4 times itself (from half a code to one) and a second moment down to
    # 1.5^-4: the second step is at most lr (0.9 * 4 + 1) * 0.1 / 0.19 / sqrt((0.999 * 1.5^-4 + 1) * 0.001 / 0.001999) = 3.2 lr.
    assert ((p[3 * BLOCK:4 * BLOCK] - 1).abs() <= 4.2e-2).all()


def test_more_than_one_piece(gpu, monkeypatch):
    """Tensors longer than a table entry are cut: the same bits as whole."""
    from addernetcuda_amd import optim
    for bits in (32, 8):
        outs = []
        for piece in (1 << 30, 1024):
            monkeypatch.setattr(optim, "_PIECE", piece)
            ps = params(torch.float32, 5, [(5000,), (7,), (1024, 300)])
            opt = optim.AdamW(ps, lr=1e-2, state_bits=bits)
            for t in range(2):
                set_grads(ps, t)
                opt.step()
            outs.append([p.detach().clone() for p in ps] + [opt.state[p]["exp_avg"] for p in ps])
        for a, b in zip(*outs):
            assert torch.equal(a, b)


def test_a_step_is_a_change_in_place(gpu):
    from addernetcuda_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW([p], lr=0.1)
    (p * p).sum().backward()
    y = (p * p).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(gpu):
    from addernetcuda_amd import optim
    p = torch.nn.Parameter(torch.ones(5000, device="cuda"))
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([p], state_bits=4)
    with pytest.raises(ValueError, match="amsgrad"):
        optim.AdamW([p], state_bits=8, amsgrad=True)
    q = torch.nn.Parameter(torch.ones(50, 100, device="cuda").t())
    q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="state_bits=8 needs"):
        optim.AdamW([q], state_bits=8).step()
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p], state_bits=8)
    opt.step()
    opt.state[p]["exp_avg_scale"] = opt.state[p]["exp_avg_scale"][:3]
    with pytest.raises(RuntimeError, match="does not fit"):
        opt.step()
    with pytest.raises(RuntimeError, match="int8 or uint8"):
        optim.state_values(p.detach(), p.detach())
    with pytest.raises(RuntimeError, match="scales must be"):
        optim.state_values(torch.zeros(300, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        optim.state_values(torch.zeros(3, dtype=torch.int8), torch.zeros(1))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("begun", [False, True])
def test_copies_and_pickles_step_as_the_original(begun, capturable, bits, gpu):
    import pickle
    from addernetcuda_amd.optim import AdamW
    ps = params(torch.float32, 4)
    opt = AdamW(ps, lr=1e-2, state_bits=bits, min_8bit_size=300, capturable=capturable)
    if begun:
        set_grads(ps, 1)
        opt.step()
    others = [copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))]
    for o in [opt] + others:
        assert (o.state_bits, o.min_8bit_size) == (bits, 300)
        set_grads(o.param_groups[0]["params"], 2)
        o.step()
    for o in others:
        for p, q in zip(ps, o.param_groups[0]["params"]):
            assert p is not q and torch.equal(p, q)
            for name, value in opt.state[p].items():
                other = o.state[q][name]
                assert value == other if not isinstance(value, torch.Tensor) else torch.equal(value, other) and value.dtype == other.dtype
        if capturable:
            assert len({id(s["step"]) for s in o.state.values()}) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("capturable", [False, True])
def test_gradients_that_the_kernel_leaves_in_either_type(capturable, dtype, gpu):
    """One gradient that is not contiguous sends its group to torch for that step, where moments have the parameter's type; before and behind it
    the kernel's are float32.  What torch does with the same state is what comes out."""
    from addernetcuda_amd.optim import AdamW
    a = params(dtype, 3, [(40, 50), (30, 20), (700,)])
    o = AdamW(a, lr=1e-2, weight_decay=0.1, capturable=capturable)
    for t in range(6):
        set_grads(a, t)
        if t in (2, 3):
            b = [torch.nn.Parameter(p.detach().clone()) for p in a]
            r = torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1, foreach=False, capturable=capturable)
            for p, q in zip(a, b):
                q.grad = p.grad.clone()
                r.state[q] = {name: value.detach().clone().to(dtype) for name, value in o.state[p].items() if name != "step"}
                r.state[q]["step"] = torch.tensor(float(t), device="cuda" if capturable else "cpu")
            a[1].grad = a[1].grad.t().contiguous().t()
        o.step()
        assert all(float(o.state[p]["step"]) == t + 1 for p in a)
        if t in (2, 3):
            r.step()
            for p, q in zip(a, b):
                assert o.state[p]["exp_avg"].dtype == dtype and torch.equal(o.state[p]["exp_avg"], r.state[q]["exp_avg"])
                assert torch.equal(o.state[p]["exp_avg_sq"], r.state[q]["exp_avg_sq"]) and torch.equal(p, q)
        else:
            assert all(o.state[p]["exp_avg"].dtype == torch.float32 for p in a)


@pytest.mark.parametrize("kind", ["foreach", "fused"])
def test_a_state_of_torchs_other_steps_goes_both_ways(kind, gpu):
    """The state of torch's fused or foreach optimizer is taken on by the kernel, and by torch for a gradient that the kernel leaves."""
    from addernetcuda_amd.optim import AdamW
    shapes = [(40, 50), (30, 20)]
    a, b = params(torch.float32, 3, shapes), params(torch.float32, 3, shapes)
    r = torch.optim.AdamW(b, lr=1e-2, **{kind: True})
    for t in range(5):
        for ps in (a, b):
            set_grads(ps, t)
        r.step()
        if t == 0:
            o = AdamW(a, lr=1e-2)
            o.load_state_dict(copy.deepcopy(r.state_dict()))
            with torch.no_grad():
                for p, q in zip(a, b):
                    p.copy_(q)
            continue
        if t == 2:
            a[1].grad = a[1].grad.t().contiguous().t()
        o.step()
        for p, q in zip(a, b):
            assert torch.allclose(p, q, rtol=1e-6, atol=1e-6), t


def test_counts_that_part_are_as_few_as_they_differ(gpu):
    """Parameters that stay behind together share one count; a step that torch takes leaves the counts shared; all of them are right, also in a
    captured step that torch takes."""
    from addernetcuda_amd.optim import AdamW
    ps = params(torch.float32, 3, [(40, 50)] * 6)
    opt = AdamW(ps, lr=1e-3, capturable=True)
    count = lambda: (len({id(opt.state[p]["step"]) for p in ps}), [int(opt.state[p]["step"]) for p in ps])

    def step(which, across=False, keep=False):
        if not keep:
            set_grads(ps, 1)
            for i, p in enumerate(ps):
                p.grad = None if i not in which else p.grad.t().contiguous().t() if across else p.grad
        opt.step()

    step(range(6))
    assert count() == (1, [1] * 6)
    step(range(3))
    assert count() == (2, [2, 2, 2, 1, 1, 1])
    step(range(3, 6))
    assert count() == (2, [2] * 6)
    step(range(6), across=True)
    assert count() == (2, [3] * 6)
    step(range(6))
    assert count() == (2, [4] * 6)
    step((0, 1, 3), across=True)
    assert count() == (4, [5, 5, 4, 5, 4, 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(range(6), across=True)
        assert count() == (4, [6, 6, 5, 6, 5, 5])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(range(6), keep=True)
    torch.cuda.current_stream().wait_stream(side)
    for t in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert count() == (4, [7 + t, 7 + t, 6 + t, 7 + t, 6 + t, 6 + t])
    step(range(6))
    assert count() == (4, [10, 10, 9, 10, 9, 9])
    plain = AdamW(ps, lr=1e-3)   # a state that counted on the host, and from now on on the device
    set_grads(ps, 5)
    plain.step()
    plain.param_groups[0]["capturable"] = True
    plain.step()
    assert len({id(plain.state[p]["step"]) for p in ps}) == 1 and int(plain.state[ps[0]]["step"]) == 2


@pytest.mark.parametrize("begun", [False, True])
def test_a_captured_step_needs_its_count_on_the_device(begun, gpu):
    """As torch's own optimizer: a count on the host would be frozen into the graph."""
    from addernetcuda_amd.optim import AdamW
    ps = params(torch.float32, 3, [(40, 50), (7,)])
    opt = AdamW(ps, lr=1e-3)
    set_grads(ps, 1)
    if begun:
        opt.step()
    before = [p.detach().clone() for p in ps]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capturable=True"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps, before)) and len(opt.state) == (len(ps) if begun else 0)
    opt.step()
    assert all(opt.state[p]["step"] == 1 + begun for p in ps)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_workgroups_than_one_launch_takes(bits, gpu, monkeypatch):
    """Tensors that are too many values for one launch together go into several: the same bits as in one."""
    from addernetcuda_amd import optim
    outs = []
    for groups in (optim._GROUPS, 3, 1):
        monkeypatch.setattr(optim, "_GROUPS", groups)
        ps = params(torch.float32, 5, [(5000,), (7,), (1024, 2), (1024,), (3,), (2000,), (9, 9)])
        opt = optim.AdamW(ps, lr=1e-2, state_bits=bits, min_8bit_size=600)
        for t in range(2):
            set_grads(ps, t)
            opt.step()
        outs.append([p.detach().clone() for p in ps] + [opt.state[p]["exp_avg"] for p in ps])
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)
