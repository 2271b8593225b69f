"""GPU: the dense product in 8-bit integers against its definition.

Scales and integers have to be equal to those of 64-bit arithmetic.  The outputs are an exact integer
times two float32 scales: one rounding for the integer (2^-24), two for the factors (2^-24 each), and
half a step of a 16-bit output type.  Every output is held to that, relative to its own value.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def quantized(x):
    """Rows of a CPU tensor: ``(integers, scales)`` in 64 bits, by the definition."""
    x = x.double()
    scale = (x.abs().amax(-1) / 127).float().double()
    return (x / torch.where(scale > 0, scale, 1.).unsqueeze(-1)).round(), scale


def make(M, K, N, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen) * torch.exp(torch.randn(M, 1, generator=gen))
    w = torch.randn(K, N, generator=gen) * torch.exp(torch.randn(1, N, generator=gen)) * K ** -0.5
    return x.to(dtype), w


def close(y, want, dtype):
    step = 3 * 2 ** -24 + (torch.finfo(dtype).eps / 2 if dtype != F32 else 0)
    y, want = y.cpu().double(), want.double()
    assert y.shape == want.shape and bool((torch.isnan(y) == torch.isnan(want)).all())
    least = 2 ** -25 if dtype == F16 else 0        # half a step among the subnormal numbers
    assert bool((((y - want).abs() <= step * 1.001 * want.abs() + least) | torch.isnan(want)).all())


# rows on both sides of every change of kernel and tile (4, 8, 16, 24, 32 | 64, 128, 256), channels likewise; rows that a
# product's blocks quantise themselves (up to 4 x 40704 bytes in all)
SIZES = [(2, 1000, 40), (3, 8192, 33), (3, 77, 64), (4, 4096, 100), (4, 10176, 20), (4, 10192, 20), (1, 40704, 16), (1, 40720, 17),
         (5, 513, 30), (1, 16, 1), (1, 1000, 17), (7, 64, 16), (8, 100, 33), (9, 4096, 70), (16, 31, 16), (17, 1, 40), (24, 640, 48),
         (31, 257, 100), (32, 2048, 65), (33, 64, 64), (64, 500, 129), (127, 128, 256), (128, 129, 255), (129, 4096, 300),
         (100, 8192, 520), (40, 16000, 64), (200, 1001, 777), (1000, 96, 1000)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('M,K,N', SIZES)
def test_product(cuda, dtype, M, K, N):
    from brainstate_b200 import quant
    x, w = make(M, K, N, dtype, seed=M + K)
    w8 = quant.Int8Dense(w.cuda())
    wq, ws = quantized(w.t())
    assert torch.equal(w8.q[:, :K].cpu().double(), wq) and torch.equal(w8.scale.cpu().double(), ws)
    assert not w8.q[:, K:].any()
    rows = quant.quantize_rows(x.cuda())
    xq, xs = quantized(x)
    assert torch.equal(rows.q[:, :K].cpu().double(), xq) and torch.equal(rows.scale.cpu().double(), xs)
    assert not rows.q[:, K:].any()
    want = (xq @ wq.t()) * xs.unsqueeze(1) * ws
    y = x.cuda() @ w8
    assert y.dtype == dtype
    close(y, want, dtype)
    assert torch.equal(rows @ w8, y)
    assert torch.equal(rows.dequantize().cpu(), (xq * xs.unsqueeze(1)).float())
    assert torch.equal(w8.dequantize().cpu(), (wq * ws.unsqueeze(1)).float().t())
    close(quant.int8_matmul(x.cuda(), w8, out_dtype=F32), want, F32)


@pytest.mark.parametrize('M,N', [(1, 300), (300, 1000), (2000, 2048)])
@pytest.mark.parametrize('kind', ['bool', 'uint8', 'float32'])
def test_spikes(cuda, M, N, kind):
    """Spikes enter as 0 and 1 whatever number marks them; bit for bit like the sum of the dequantised rows in 64 bits."""
    from brainstate_b200 import EventArray, quant
    K = 1203
    gen = torch.Generator().manual_seed(M)
    spk = torch.rand(M, K, generator=gen) < 0.1
    spk[M // 2] = False
    w = torch.randn(K, N, generator=gen)
    marked = {'bool': spk, 'uint8': spk.to(torch.uint8) * 7, 'float32': spk.float() * -2.5}[kind]
    w8 = quant.Int8Dense(w.cuda())
    wq, ws = quantized(w.t())
    y = EventArray(marked.cuda()) @ w8
    assert y.dtype == F32
    assert torch.equal(y.cpu(), ((spk.double() @ wq.t()).float() * ws.float()))


def test_many_tiles_per_block(cuda):
    """More tiles than blocks, wide ones: the ring and both halves of tensor memory go round many times."""
    from brainstate_b200 import quant
    gen = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randn(2500, 1100, generator=gen, device='cuda')
    w8 = quant.Int8Dense(torch.randn(1100, 9000, generator=gen, device='cuda'))
    rows = quant.quantize_rows(x)
    want = (rows.q[:, :1100].double() @ w8.q[:, :1100].t().double()) * rows.scale.double().unsqueeze(1) * w8.scale.double()
    y = rows @ w8
    close(y, want.cpu(), F32)
    assert all(torch.equal(rows @ w8, y) for _ in range(3))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_ties_and_borders(cuda, dtype):
    """Values exactly between two integers go to the even one, their neighbours to their own side."""
    from brainstate_b200 import quant
    rows = []
    for top in (127., 254., 1., 3.7e-3):
        s = torch.tensor(top, dtype=dtype).float() / 127
        half = ((torch.arange(-126, 126) + 0.5) * s).to(dtype)
        up = torch.nextafter(half.float(), torch.tensor(1e9)).to(dtype)
        down = torch.nextafter(half.float(), torch.tensor(-1e9)).to(dtype)
        rows.append(torch.cat([torch.tensor([top]).to(dtype), half, up, down]))
    x = torch.stack(rows)
    got = quant.quantize_rows(x.cuda())
    q, s = quantized(x)
    assert torch.equal(got.scale.cpu().double(), s) and torch.equal(got.q[:, :x.shape[1]].cpu().double(), q)


@pytest.mark.parametrize('M', [5, 200])
def test_rows_and_channels_without_a_scale(cuda, M):
    """Zero rows and channels give zeros; rows and channels with NaN or infinity give NaN and spoil nothing else; huge
    and tiny rows keep their values."""
    from brainstate_b200 import quant
    x, w = make(M, 72, 50, F32, seed=1)
    x[0] = 0
    x[1, 3] = float('nan')
    x[2, 71] = float('-inf')
    x[3] *= 1e37 / x[3].abs().max()
    x[4] *= 1e-36 / x[4].abs().max()
    w[:, 7] = 0
    w[0, 9] = float('inf')
    w[71, 11] = float('nan')
    y = (x.cuda() @ quant.Int8Dense(w.cuda())).cpu()
    bad = torch.zeros(M, 50, dtype=torch.bool)
    bad[1:3] = True
    bad[:, [9, 11]] = True
    assert torch.equal(torch.isnan(y), bad)
    wf, xf = torch.where(torch.isfinite(w), w, 0.), torch.where(torch.isfinite(x), x, 0.)
    wq, ws = quantized(wf.t())
    xq, xs = quantized(xf)
    want = (xq @ wq.t()) * xs.unsqueeze(1) * ws
    # results below 2^-126 lie 2^-149 apart: half of that for their rounding
    far = (y.double() - want).abs() > 3.01 * 2 ** -24 * want.abs() + 2 ** -150
    assert not far[~bad].any() and not y[0, :9].any() and not y[5:, 7].any()


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_strides_and_leading_dimensions(cuda, dtype):
    from brainstate_b200 import quant
    x, w = make(60, 96, 40, dtype)
    w8 = quant.Int8Dense(w.cuda())
    xc = x.cuda()
    want = xc @ w8
    assert torch.equal(xc.reshape(3, 4, 5, 96) @ w8, want.reshape(3, 4, 5, 40))
    assert torch.equal(xc[0] @ w8, want[0])
    wide = torch.zeros(60, 200, device='cuda', dtype=dtype)
    for off in (0, 3, 8):                       # rows of a wider tensor, at offsets of every alignment
        wide[:, off:off + 96] = xc
        assert torch.equal(wide[:, off:off + 96] @ w8, want)
    assert torch.equal(xc.t().contiguous().t() @ w8, want)
    assert torch.equal(quant.Int8Dense(w.t().contiguous().t().cuda()).q, w8.q)
    assert torch.equal(xc[:1].expand(50, 96) @ w8, want[:1].expand(50, 40))
    assert (xc[:0] @ w8).shape == (0, 40) and (xc.reshape(5, 12, 96)[:, :0] @ w8).shape == (5, 0, 40)


def test_streams_and_graphs(cuda):
    """On a side stream, and captured: two graphs of both kernels replayed in turn on changed inputs."""
    from brainstate_b200 import quant
    x, w = make(40, 5000, 64, BF16)
    w8 = quant.Int8Dense(w.cuda())
    xs = x.cuda()
    want = xs @ w8, xs[:3] @ w8
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = xs @ w8, xs[:3] @ w8
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = xs @ w8
    with torch.cuda.graph(g2):
        y2 = xs[:3] @ w8
    for f in (1., -3.):
        xs.copy_(x.cuda() * f)
        g1.replay(); g2.replay(); g1.replay()
        assert torch.equal(y1, xs @ w8) and torch.equal(y2, xs[:3] @ w8)


def test_layer_and_projections_of_a_plastic_synapse(cuda):
    """As they are used: a trained dense layer is quantised and serves, and its products feed a synapse that learns; one
    quantisation of the input serves all projections; steps agree with the whole sequence."""
    from brainstate_b200 import EventArray, nn, quant, plastic
    torch.manual_seed(3)
    B, T, H, d, n = 3, 33, 2, 16, 120
    layer = nn.EventLinear(n, 2 * H * d, lambda shape: torch.randn(shape).numpy() * n ** -0.5, float_as_event=False)
    int8 = layer.quantized()
    x = torch.randn(B, T, n, device='cuda')
    full = layer(x)
    assert (int8(x) - full).norm() < 0.02 * full.norm()
    events = nn.EventLinear(n, 3 * H, lambda shape: torch.randn(shape).numpy() * n ** -0.5).quantized()
    spk = x > 1.5
    assert torch.equal(events(spk), EventArray(spk) @ events.weight)
    wv, wg = (quant.Int8Dense(torch.randn(n, m, device='cuda') * n ** -0.5) for m in (H * d, 2 * H))

    def project(x):
        rows = quant.quantize_rows(x)
        q, k = int8(x).unflatten(-1, (2, H, d)).unbind(-3)
        v = (rows @ wv).unflatten(-1, (H, d))
        g, beta = (rows @ wg).unflatten(-1, (2, H)).unbind(-2)
        return q, torch.nn.functional.normalize(k, dim=-1), v, -torch.nn.functional.softplus(g), torch.sigmoid(beta)

    o, state = plastic.delta_rule(*project(x))
    synapse = nn.DeltaSynapse(d, d, k_heads=H)
    synapse.init_state(B)
    steps = torch.stack([synapse(*project(x[:, t])) for t in range(T)], 1)
    # same integers and sums in both kernels of the product: the projections are equal; the rule's two forms to 1e-5
    assert (steps - o).norm() <= 1e-5 * o.norm() and (synapse.state.value - state).norm() <= 1e-5 * state.norm()


def test_refusals(cuda):
    from brainstate_b200 import EventArray, nn, quant
    x, w = make(4, 32, 16, F32)
    w8 = quant.Int8Dense(w.cuda())
    xc = x.cuda()
    with pytest.raises(ValueError, match='rows of 32'):
        xc[:, :31] @ w8
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        xc.double() @ w8
    with pytest.raises(TypeError, match='spikes'):
        EventArray(xc.half()) @ w8
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        x @ w8
    with pytest.raises(RuntimeError, match='no gradient'):
        xc.clone().requires_grad_(True) @ w8
    with torch.no_grad():
        assert torch.equal(xc.clone().requires_grad_(True) @ w8, xc @ w8)
    with pytest.raises(ValueError, match='must be'):
        quant.Int8Dense(xc[0])
    with pytest.raises(ValueError, match='without inputs'):
        quant.Int8Dense(torch.zeros(0, 4, device='cuda'))
    with pytest.raises(TypeError, match='out_dtype'):
        quant.int8_matmul(xc, w8, out_dtype=torch.float64)
    with pytest.raises(ValueError, match='rows of 32, expected 16'):
        quant.quantize_rows(xc) @ quant.Int8Dense(torch.zeros(16, 4, device='cuda'))
    with pytest.raises(RuntimeError, match='131072'):
        quant.Int8Dense(torch.zeros(131073, 1, device='cuda'))
    with pytest.raises(ValueError, match='one weight'):
        nn.EventLinear(4, 4, 0.5).quantized()
