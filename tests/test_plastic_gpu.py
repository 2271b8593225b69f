"""GPU: the gated delta rule against its definition in 64 bits.

Tolerances (2-norm of the error over that of the result).  A product of two 32-bit operands drops
lo x lo (2^-22) and cuts lo (2^-21 of the operand); its sums over at most 128 terms pass through
at most 48 tensor instructions that cut the running sum (2^-24 each on average, relative to a sum that
grows towards its final size, so half of that): 48 * 2^-25 + 2^-21 + 2^-22 = 2.2e-6.  At most four such
products follow each other between an input and a 32-bit result: 32-bit results are held to 1e-5.
A 16-bit result adds half a step of its type; bf16 results also the rounding of one operand of the
last product to tf32 (2^-12, P of both: 2^-11).
"""
import pytest
import torch

from plastic_reference import delta_rule as reference
from plastic_reference import error, inputs

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tolerance(dtype):
    if dtype == F32:
        return 1e-5
    return torch.finfo(dtype).eps / 2 + 1e-5 + (2 ** -11 if dtype == BF16 else 0)


def run_both(args, lengths=None, scale=None, grads=True, seed=5):
    """Outputs and gradients of the kernels and of the definition, by name."""
    from brainstate_b200 import plastic
    scale = args['q'].shape[-1] ** -0.5 if scale is None else scale
    ref = {n: x.double().requires_grad_(grads) for n, x in args.items()}
    dev = {n: x.cuda().requires_grad_(grads) for n, x in args.items()}
    rl = None if lengths is None else torch.tensor(lengths)
    dl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    ro, rs = reference(*(ref[n] for n in ('q', 'k', 'v', 'g', 'beta')), scale, ref.get('initial'), rl)
    o, s = plastic.delta_rule(*(dev[n] for n in ('q', 'k', 'v', 'g', 'beta')), scale=scale,
                              initial_state=dev.get('initial'), lengths=dl)
    assert o.dtype == args['v'].dtype and s.dtype == F32
    got, want = {'o': o, 'state': s}, {'o': ro, 'state': rs}
    if grads:
        gen = torch.Generator().manual_seed(seed)
        do = torch.randn(ro.shape, generator=gen, dtype=torch.float64).to(args['v'].dtype)
        ds = (0.3 * torch.randn(rs.shape, generator=gen, dtype=torch.float64)).float()
        names = list(args)
        rg = torch.autograd.grad((ro, rs), [ref[n] for n in names], (do.double(), ds.double()), allow_unused=True)
        dg = torch.autograd.grad((o, s), [dev[n] for n in names], (do.cuda(), ds.cuda()))
        for n, x, y in zip(names, dg, rg):
            assert x.dtype == args[n].dtype and x.shape == args[n].shape
            got['d' + n], want['d' + n] = x, torch.zeros(args[n].shape, dtype=torch.float64) if y is None else y
    return got, want


def compare(got, want):
    far = {n: (error(got[n], want[n]), tolerance(got[n].dtype)) for n in want}
    assert all(e <= t for e, t in far.values()), far


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('T', [1, 2, 8, 9, 16, 63, 64, 65, 200])
def test_lengths(cuda, dtype, T):
    compare(*run_both(inputs(2, T, 2, 2, 64, 48, dtype, seed=T)))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('dk,dv', [(1, 1), (16, 20), (33, 100), (64, 16), (65, 33), (100, 192), (128, 128), (128, 300), (8, 1100)])
def test_sizes(cuda, dtype, dk, dv):
    compare(*run_both(inputs(1, 150, 1, 2, dk, dv, dtype, seed=dk)))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('B,Hk,Hv,dk', [(5, 3, 9, 128), (20, 4, 8, 64), (24, 4, 8, 128), (1, 1, 1, 128)])
def test_heads_and_batches(cuda, dtype, B, Hk, Hv, dk):
    """Grids of every division of the value columns among warps and blocks."""
    compare(*run_both(inputs(B, 70, Hk, Hv, dk, 128, dtype, seed=B)))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('T', [7, 9, 130])
def test_padded_rows(cuda, dtype, T):
    """What lies behind a row's length is not read (it holds NaN and infinities here), and comes out as zero."""
    args = inputs(5, T, 2, 4, 48, 40, dtype, seed=T)
    lengths = [0, 1, T, T // 2, max(T - 1, 0)]
    for b, n in enumerate(lengths):
        for name, bad in (('q', float('nan')), ('k', float('inf')), ('v', float('nan')), ('g', float('-inf')),
                          ('beta', float('nan'))):
            args[name][b, n:] = bad
    got, want = run_both(args, lengths)
    compare(got, want)
    for b, n in enumerate(lengths):
        for name in ('o', 'dq', 'dk', 'dv', 'dg', 'dbeta'):
            assert torch.all(got[name][b, n:] == 0), name
    assert torch.equal(got['state'][0].cpu(), args['initial'][0])


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('T,Hk,dk,dv', [(8, 2, 48, 40), (200, 1, 64, 48), (200, 2, 33, 20), (130, 2, 128, 132), (129, 1, 7, 9)])
def test_everything_behind_a_length_is_written(cuda, dtype, T, Hk, dk, dv):
    """With new memory full of NaN: outputs and gradients behind a length are zero, all others are finite and right."""
    args = inputs(6, T, Hk, 2, dk, dv, dtype, seed=T + dk)
    lengths = [0, 1, min(64, T), min(65, T), T - 1, T]
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)       # fills what is allocated without a value
    try:
        assert torch.empty(64, device='cuda').isnan().all()
        got, want = run_both(args, lengths)
    finally:
        torch.use_deterministic_algorithms(before)
    compare(got, want)
    for b, n in enumerate(lengths):
        for name in ('o', 'dq', 'dk', 'dv', 'dg', 'dbeta'):
            assert torch.all(got[name][b, n:] == 0), name


def test_lengths_out_of_range_are_clipped(cuda):
    from brainstate_b200 import plastic
    args = {n: x.cuda() for n, x in inputs(3, 40, 1, 1, 16, 16, F32).items()}
    initial = args.pop('initial')
    run = lambda n: plastic.delta_rule(*args.values(), initial_state=initial, lengths=torch.tensor(n, device='cuda'))
    for x, y in zip(run([-5, 2 ** 40, 40]), run([0, 40, 40])):
        assert torch.equal(x, y)


@pytest.mark.parametrize('T', [7, 10, 140])
def test_full_decay_and_no_learning(cuda, T):
    """g = -inf drops the state, large decays and beta = 0 and 1 in between; nothing turns into NaN."""
    args = inputs(2, T, 1, 2, 32, 32, F32, seed=3)
    args['g'][:, T // 3] = float('-inf')
    args['g'][0, T // 2] = -500.
    args['g'][1, T // 2:T // 2 + 3] = -60.
    args['beta'][:, ::4] = 0.
    args['beta'][:, 1::4] = 1.
    got, want = run_both(args)
    # the definition's own gradient at -inf is e^g times something finite: zero
    assert all(torch.isfinite(x).all() for x in got.values())
    want['dg'] = torch.nan_to_num(want['dg'])
    compare(got, want)


def test_alike_keys(cuda):
    """Keys of a chunk that are nearly the same: (I + A)^{-1} must not be summed as a power series."""
    args = inputs(1, 128, 1, 1, 64, 64, F32, seed=8, alike=6.0)
    compare(*run_both(args))


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_long_sequence(cuda, dtype):
    """3000 tokens (47 chunks) with slow decay: errors must not pile up from chunk to chunk."""
    args = inputs(1, 3000, 1, 2, 16, 16, dtype, seed=12)
    args['g'] *= 0.05
    compare(*run_both(args))


def test_many_rows_of_different_length(cuda):
    """More chunks than the reverse kernel has blocks, most rows short: chunks are handed out as blocks become free."""
    args = inputs(60, 200, 2, 4, 16, 16, F32, seed=9)
    compare(*run_both(args, [(7 * b) % 201 if b % 3 else b % 5 for b in range(60)]))


def test_two_streams_at_once(cuda):
    """Two calls in flight with workspaces of their own, rows of different length among them."""
    from brainstate_b200 import plastic
    sets = []
    for seed in (1, 2):
        a = {n: x.cuda() for n, x in inputs(9, 260, 2, 4, 64, 64, BF16, seed=seed).items()}
        sets.append((a.pop('initial'), [x.requires_grad_(True) for x in a.values()],
                     torch.arange(9, device='cuda', dtype=torch.int32) * 32))

    def once(initial, leaves, lengths):
        o, s = plastic.delta_rule(*leaves, initial_state=initial, lengths=lengths)
        return (o, s) + torch.autograd.grad(o.float().square().sum() + s.sum(), leaves)

    want = [once(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(once(*x))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_zero_tokens_and_empty_batch(cuda):
    from brainstate_b200 import plastic
    z = lambda *s: torch.zeros(*s, device='cuda')
    initial = torch.randn(2, 4, 8, 8, device='cuda', requires_grad=True)
    o, s = plastic.delta_rule(z(2, 0, 2, 8), z(2, 0, 2, 8), z(2, 0, 4, 8), z(2, 0, 4), z(2, 0, 4), initial_state=initial)
    assert o.shape == (2, 0, 4, 8) and torch.equal(s, initial)
    ct = torch.randn_like(s)
    assert torch.equal(torch.autograd.grad(s, initial, ct)[0], ct)
    o, s = plastic.delta_rule(z(0, 5, 2, 8), z(0, 5, 2, 8), z(0, 5, 4, 8), z(0, 5, 4), z(0, 5, 4))
    assert o.shape == (0, 5, 4, 8) and s.shape == (0, 4, 8, 8)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('T', [5, 80])
def test_strides_and_alignment(cuda, dtype, T):
    """Views of one fused projection, an odd offset, a broadcast gate and a dense-last copy give the dense result."""
    from brainstate_b200 import plastic
    B, H, d = 2, 2, 32
    fused = torch.randn(B, T, 3 * H * d + 1, device='cuda', dtype=dtype)
    for off in (0, 1):
        q, k, v = (fused[..., off + i * H * d:off + (i + 1) * H * d].unflatten(-1, (H, d)) for i in range(3))
        k = torch.nn.functional.normalize(k.float(), dim=-1).to(dtype).transpose(1, 2).contiguous().transpose(1, 2)
        g = torch.full((1, 1, H), -0.1, device='cuda').expand(B, T, H)
        beta = torch.rand(H, T, B, device='cuda').permute(2, 1, 0)
        got = plastic.delta_rule(q, k, v, g, beta)
        want = plastic.delta_rule(*(x.contiguous().clone() for x in (q, k, v, g, beta)))
        # the copies may take the wide loads: same values, same order of sums
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    t = torch.randn(B, T, d, H, device='cuda', dtype=dtype).transpose(2, 3)      # last dimension not dense
    assert torch.equal(plastic.delta_rule(t, k, v, g, beta)[0], plastic.delta_rule(t.contiguous(), k, v, g, beta)[0])


def test_broadcast_inputs_and_casts_have_gradients(cuda):
    from brainstate_b200 import plastic
    a = {n: x.cuda() for n, x in inputs(2, 40, 1, 2, 16, 16, F32, state=False).items()}
    rate = torch.tensor(0.4, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    full = torch.full((2, 40, 2), 0.4, device='cuda', dtype=torch.bfloat16).float().requires_grad_(True)
    o1, _ = plastic.delta_rule(a['q'], a['k'], a['v'], a['g'], rate.expand(2, 40, 2))
    o2, _ = plastic.delta_rule(a['q'], a['k'], a['v'], a['g'], full)
    assert torch.equal(o1, o2)
    g1, = torch.autograd.grad(o1.square().sum(), rate)
    g2, = torch.autograd.grad(o2.square().sum(), full)
    assert g1.dtype == torch.bfloat16
    assert abs(float(g1) - float(g2.sum())) <= 2 ** -8 * 1.01 * float(g2.abs().sum())


def test_gradients_against_differences(cuda):
    """Along random directions: central differences of the kernels' own 32-bit results.  A step of 1e-2 leaves a
    third-order term of about 1e-4 and rounding of about 1e-6 / 1e-2."""
    from brainstate_b200 import plastic
    args = {n: x.cuda() for n, x in inputs(1, 90, 1, 2, 32, 24, F32, seed=4).items()}
    names = list(args)
    wo, ws = torch.randn(1, 90, 2, 24, device='cuda'), torch.randn(1, 2, 32, 24, device='cuda')

    def f(xs):
        o, s = plastic.delta_rule(*xs[:5], initial_state=xs[5])
        return (o * wo).double().sum() + (s * ws).double().sum()

    xs = [args[n].requires_grad_(True) for n in names]
    grads = torch.autograd.grad(f(xs), xs)
    torch.manual_seed(1)
    for i, n in enumerate(names):
        d = torch.randn_like(xs[i])
        d = d / d.norm() * xs[i].detach().norm()
        h = 1e-2
        with torch.no_grad():
            up = f([x + h * d if j == i else x for j, x in enumerate(xs)])
            down = f([x - h * d if j == i else x for j, x in enumerate(xs)])
        diff, want = float((up - down) / (2 * h)), float((grads[i] * d).double().sum())
        assert abs(diff - want) <= 5e-3 * float(grads[i].norm() * d.norm()), (n, diff, want)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('B,Hk,Hv,dk,dv', [(1, 1, 1, 1, 1), (3, 2, 4, 33, 20), (2, 2, 2, 64, 64), (5, 1, 3, 128, 132),
                                           (70, 2, 4, 128, 128), (400, 2, 4, 128, 128), (601, 1, 2, 64, 36),
                                           (310, 2, 4, 113, 128), (300, 1, 4, 128, 112), (1200, 1, 1, 16, 16)])
def test_steps_in_place(cuda, dtype, B, Hk, Hv, dk, dv):
    """Several single steps: each output and the last state against the definition, and the state tensor is the same."""
    from brainstate_b200 import plastic
    T = 4
    args = inputs(B, T, Hk, Hv, dk, dv, dtype, seed=dk)
    ro, rs = reference(*(args[n].double() for n in ('q', 'k', 'v', 'g', 'beta')), 0.7, args['initial'].double())
    state = args['initial'].cuda()
    version = state._version
    at = state.data_ptr()
    for t in range(T):
        o = plastic.delta_rule_step(*(args[n][:, t].cuda() for n in ('q', 'k', 'v', 'g', 'beta')), state, scale=0.7)
        assert error(o, ro[:, t]) <= tolerance(dtype)
    assert error(state, rs) <= 1e-5 and state.data_ptr() == at and state._version == version + T


def test_step_sees_the_previous_step_of_the_layer(cuda):
    """The layer: steps in place, steps with gradients and one sequence give the same."""
    from brainstate_b200 import nn
    args = {n: x.cuda() for n, x in inputs(2, 20, 1, 2, 16, 24, F32, state=False).items()}
    layer = nn.DeltaSynapse(16, 24, k_heads=1, v_heads=2)
    with pytest.raises(RuntimeError, match='init_state'):
        layer(*(x[:, 0] for x in args.values()))
    layer.init_state(2)
    steps = torch.stack([layer(*(x[:, t] for x in args.values())) for t in range(20)], 1)
    stepped = layer.state.value
    layer.reset_state(2)
    seq = layer.run(*args.values())
    assert error(seq, steps.cpu()) <= 1e-5 and error(layer.state.value, stepped.cpu()) <= 1e-5
    layer.reset_state(2)
    v = args['v'].clone().requires_grad_(True)
    outs = torch.stack([layer(*(dict(args, v=v)[n][:, t] for n in args)) for t in range(20)], 1)
    g1, = torch.autograd.grad(outs.square().sum(), v)
    layer.reset_state(2)
    g2, = torch.autograd.grad(layer.run(*dict(args, v=v).values()).square().sum(), v)
    assert error(g1, g2.cpu()) <= 2e-5


def test_results_do_not_vary_and_streams(cuda):
    """Same bits on every call, also from another stream than the default one while it is busy."""
    from brainstate_b200 import plastic
    args = {n: x.cuda() for n, x in inputs(3, 300, 2, 6, 64, 64, BF16, seed=2).items()}
    initial = args.pop('initial')
    leaves = [x.requires_grad_(True) for x in args.values()]

    def once():
        o, s = plastic.delta_rule(*leaves, initial_state=initial)
        return (o, s) + torch.autograd.grad((o.float().sum() + s.sum()), leaves)

    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    third = once()
    torch.cuda.synchronize()
    for x, y, z in zip(first, second, third):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_captured_and_replayed(cuda):
    """Forward and backward in one graph and a step in another, replayed with new inputs, in turn."""
    from brainstate_b200 import plastic
    a = {n: x.cuda() for n, x in inputs(2, 100, 2, 4, 32, 32, BF16, seed=1).items()}
    b = {n: x.cuda() for n, x in inputs(2, 100, 2, 4, 32, 32, BF16, seed=2).items()}
    static = {n: x.clone().requires_grad_(True) for n, x in a.items()}
    state = a['initial'].clone()

    def train(x):
        o, s = plastic.delta_rule(*(x[n] for n in ('q', 'k', 'v', 'g', 'beta')), initial_state=x['initial'])
        return (o, s) + torch.autograd.grad((o, s), list(x.values()), (torch.ones_like(o), torch.ones_like(s)))

    def step(x, s):
        return plastic.delta_rule_step(*(x[n].detach()[:, 0] for n in ('q', 'k', 'v', 'g', 'beta')), s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(static)
        step(static, state)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        outs = train(static)
    with torch.cuda.graph(g2):
        so = step(static, state)
    for data in (b, a):
        with torch.no_grad():
            for n in static:
                static[n].copy_(data[n])
            state.copy_(data['initial'])
        g1.replay()
        g2.replay()
        g1.replay()
        want = train({n: x.clone().requires_grad_(True) for n, x in data.items()})
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
        s2 = data['initial'].clone()
        assert torch.equal(so, step(data, s2)) and torch.equal(state, s2)


def test_unused_outputs(cuda):
    """Gradients through the output alone and through the state alone."""
    args = inputs(1, 70, 1, 1, 16, 16, F32, seed=6)
    from brainstate_b200 import plastic
    for which in (0, 1):
        ref = [x.double().requires_grad_(True) for x in args.values()]
        dev = [x.cuda().requires_grad_(True) for x in args.values()]
        r = reference(*ref[:5], 0.25, ref[5])[which]
        y = plastic.delta_rule(*dev[:5], scale=0.25, initial_state=dev[5])[which]
        rg = torch.autograd.grad(r.sum(), ref, allow_unused=True)
        for x, z in zip(torch.autograd.grad(y.sum(), dev), rg):
            assert error(x, torch.zeros(x.shape, dtype=torch.float64) if z is None else z) <= 1e-5


def test_second_derivatives_are_refused(cuda):
    from brainstate_b200 import plastic
    args = {n: x.cuda().requires_grad_(True) for n, x in inputs(1, 20, 1, 1, 8, 8, F32).items()}
    o, _ = plastic.delta_rule(*list(args.values())[:5])
    g, = torch.autograd.grad(o.sum(), args['v'], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_saved_state_is_guarded(cuda):
    """A state that a later step overwrites in place cannot be used by an earlier backward pass."""
    from brainstate_b200 import plastic
    args = {n: x.cuda() for n, x in inputs(1, 20, 1, 1, 8, 8, F32).items()}
    state = args.pop('initial')
    v = args['v'].requires_grad_(True)
    o, _ = plastic.delta_rule(*args.values(), initial_state=state)
    with torch.no_grad():
        plastic.delta_rule_step(*(x[:, 0] for x in args.values()), state)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        o.sum().backward()


def test_inference_mode(cuda):
    """Serving: states made inside and outside of inference mode."""
    from brainstate_b200 import nn, plastic
    args = {n: x.cuda() for n, x in inputs(2, 20, 1, 2, 16, 16, F32).items()}
    initial = args.pop('initial')
    want, state = plastic.delta_rule(*args.values(), initial_state=initial)
    outside = initial.clone()
    with torch.inference_mode():
        o, s = plastic.delta_rule(*args.values(), initial_state=initial)
        assert torch.equal(o, want) and torch.equal(s, state)
        inside = initial.clone()
        for st in (inside, outside):
            y = plastic.delta_rule_step(*(x[:, 0] for x in args.values()), st)
            assert error(y, want[:, 0].cpu()) <= 1e-5
        assert torch.equal(inside, outside)
        layer = nn.DeltaSynapse(16, 16, v_heads=2)
        layer.init_state(2)
        layer(*(x[:, 0] for x in args.values()))


def test_refusals_on_device_tensors(cuda):
    from brainstate_b200 import plastic
    a = {n: x.cuda() for n, x in inputs(2, 20, 2, 4, 8, 8, F32).items()}
    call = lambda **kw: plastic.delta_rule(*({**a, **kw}[n] for n in ('q', 'k', 'v', 'g', 'beta')),
                                           initial_state=kw.get('initial'), lengths=kw.get('lengths'))
    with pytest.raises(TypeError, match='one type'):
        call(k=a['k'].half())
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        call(q=a['q'].double(), k=a['k'].double(), v=a['v'].double())
    with pytest.raises(ValueError, match='differ in shape'):
        call(k=a['k'][:, :10])
    with pytest.raises(ValueError, match='evenly'):
        call(v=a['v'][:, :, :3], g=a['g'][..., :3], beta=a['beta'][..., :3])
    with pytest.raises(ValueError, match='must have the shape'):
        call(g=a['g'][..., :2])
    with pytest.raises(TypeError, match='floating point'):
        call(beta=a['beta'].long())
    with pytest.raises(ValueError, match='key size'):
        big = torch.zeros(2, 20, 2, 129, device='cuda')
        call(q=big, k=big)
    with pytest.raises(TypeError, match='state must be float32'):
        call(initial=a['initial'].half())
    with pytest.raises(ValueError, match='expected'):
        call(initial=a['initial'][:1])
    with pytest.raises(TypeError, match='int32 or int64'):
        call(lengths=torch.ones(2, device='cuda'))
    with pytest.raises(ValueError, match='lengths has shape'):
        call(lengths=torch.ones(3, dtype=torch.int32, device='cuda'))
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        call(lengths=torch.ones(2, dtype=torch.int32))
    one = [a[n][:, 0] for n in ('q', 'k', 'v', 'g', 'beta')]
    with pytest.raises(ValueError, match='contiguous'):
        plastic.delta_rule_step(*one, a['initial'].transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(RuntimeError, match='records no gradient'):
        plastic.delta_rule_step(one[0].clone().requires_grad_(True), *one[1:], a['initial'])
