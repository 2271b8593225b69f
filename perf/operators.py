"""Cases of the plastic and the 8-bit dense operators: real sizes, a plain form and a 64-bit form.

Operators
  ``delta_rule``       a sequence through a synaptic matrix that learns by the gated delta rule (forward, and with its
                       gradient as one training step)
  ``delta_rule_step``  one token of the same, the state updated in place
  ``int8``             rows times a dense matrix held in 8-bit integers, with a scale per row and per output channel
"""
import math

import torch

own = False
DEVICE = 'cuda'
CHUNK = 64
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------

def _delta(op, name, B, T, Hk, Hv, dk, dv, dtype, ragged=False, state=True):
    c = {'op': op, 'B': B, 'T': T, 'Hk': Hk, 'Hv': Hv, 'dk': dk, 'dv': dv, 'dtype': dtype, 'ragged': ragged,
         'state': state}
    return {'name': name, **c} if name else c


def _int8(name, M, K, N, dtype):
    c = {'op': 'int8', 'M': M, 'K': K, 'N': N, 'dtype': dtype}
    return {'name': name, **c} if name else c


def listed():
    return [
        # one stream answered token by token: latency only
        _delta('step', 'step_one_stream', 1, 1, 8, 8, 64, 64, 'bfloat16'),
        # a full server: 256 streams, two value heads per key head; the states are what moves
        _delta('step', 'step_256_streams', 256, 1, 8, 16, 128, 128, 'bfloat16'),
        # a few short sequences with sizes that fit no tile, continued from a state
        _delta('forward', 'forward_odd_f32', 3, 77, 2, 4, 48, 80, 'float32'),
        # a long prompt read in one call
        _delta('forward', 'forward_long_bf16', 1, 8192, 8, 16, 128, 128, 'bfloat16', state=False),
        # a training step on a padded batch of time series, in the framework's own type
        _delta('train', 'train_ragged_f32', 8, 500, 8, 8, 64, 64, 'float32', ragged=True),
        # a training step of ordinary size
        _delta('train', 'train_bf16', 4, 2048, 16, 16, 128, 128, 'bfloat16'),
        # one token through a trained dense layer (8192 x 4096: the dense event layer's size)
        _int8('int8_one_token', 1, 8192, 4096, 'bfloat16'),
        # the dense event layer's batch of 24 rows
        _int8('int8_24_rows_f32', 24, 8192, 4096, 'float32'),
        # sizes that fit no tile and no vector width
        _int8('int8_odd_f32', 333, 1001, 777, 'float32'),
        # spikes of a batch of trials: 0/1 rows without a scale of their own
        _int8('int8_spikes', 512, 8192, 4096, 'bool'),
        # a long prompt's projections
        _int8('int8_large_bf16', 4096, 4096, 8192, 'bfloat16'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['step', 'forward', 'train', 'int8', 'int8'])
    if kind == 'int8':
        while True:
            M, K, N = _log(rng, 1, 4096), _log(rng, 64, 8192), _log(rng, 32, 8192)
            if M * K * N <= 4096 * 4096 * 8192 and M * K * N >= 1 << 16:
                return _int8(None, M, K, N, rng.choice(['float32', 'bfloat16', 'float16', 'bool']))
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hv = Hk * rng.choice([1, 1, 2, 3])
    dk, dv = rng.choice([16, 33, 48, 64, 96, 128]), rng.choice([20, 32, 64, 80, 100, 128, 192])
    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    if kind == 'step':
        while True:
            B = _log(rng, 1, 256)
            if B * Hv * dk * dv <= 256 * 16 * 128 * 128:
                return _delta('step', None, B, 1, Hk, Hv, dk, dv, dtype)
    most = 4 * 2048 * 16 * 128 * 128 if kind == 'train' else 8192 * 16 * 128 * 128
    while True:
        B, T = _log(rng, 1, 16), _log(rng, 1, 8192 if kind == 'forward' else 2048)
        if B * T * Hv * dk * dv <= most:
            return _delta(kind, None, B, T, Hk, Hv, dk, dv, dtype, ragged=rng.random() < 0.4, state=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _unit(x):
    return x / x.square().sum(-1, keepdim=True).sqrt()


def _make(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    if case['op'] == 'int8':
        M, K, N = case['M'], case['K'], case['N']
        weight = normal(K, N) * K ** -0.5
        if case['dtype'] == 'bool':
            return {'x': uniform(M, K) < 0.05, 'weight': weight}
        # activations: rows of different sizes, a few channels larger than the rest
        x = normal(M, K) * torch.exp(0.5 * normal(M, 1)) * torch.exp(0.7 * normal(1, K))
        return {'x': x.to(TYPES[case['dtype']]), 'weight': weight}
    B, T, Hk, Hv, dk, dv = (case[n] for n in ('B', 'T', 'Hk', 'Hv', 'dk', 'dv'))
    t = TYPES[case['dtype']]
    lead = (B,) if case['op'] == 'step' else (B, T)
    # unit keys and queries (a common part makes keys of one head alike, as trained ones are), decay rates that
    # differ from head to head, learning rates in (0, 1)
    q = _unit(normal(*lead, Hk, dk)).to(t)
    k = _unit(normal(*lead, Hk, dk) + 0.5 * normal(Hk, dk)).to(t)
    v = normal(*lead, Hv, dv).to(t)
    rate = torch.exp(-5 + 4 * uniform(Hv))
    g = -rate * torch.nn.functional.softplus(normal(*lead, Hv))
    beta = torch.sigmoid(normal(*lead, Hv))
    s = {'q': q, 'k': k, 'v': v, 'g': g, 'beta': beta, 'initial': None, 'lengths': None}
    if case['op'] == 'step' or case['state']:
        s['initial'] = normal(B, Hv, dk, dv) * 0.3
    if case['ragged']:
        n = torch.randint(0, T + 1, (B,), generator=gen, device=DEVICE)
        n[0] = T
        s['lengths'] = n.to(torch.int32)
    if case['op'] == 'train':
        s['do'] = normal(B, T, Hv, dv).to(t)
        s['ds'] = normal(B, Hv, dk, dv) * 0.3
    return s


def prepare(case, seed):
    s = _make(case, seed)
    s['op'] = case['op']
    if case['op'] == 'train':
        for n in ('q', 'k', 'v', 'g', 'beta', 'initial'):
            if s[n] is not None:
                s[n].requires_grad_(True)
    if case['op'] == 'int8':
        # a server quantises its weights once
        if own:
            from brainstate_b200 import quant
            s['w8'] = quant.Int8Dense(s['weight'])
        else:
            s['wq'], s['ws'] = _plain_quantize(s['weight'].t())
            s['wq'] = s['wq'].float()
        del s['weight']
    return s


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------

def _plain_quantize(x):
    """Rows of ``x`` in 8 bits: 32-bit scales, values rounded to the nearest (ties to even; 64-bit quotients, since a
    value next to a border must fall on its side of it)."""
    top = x.abs().amax(-1).double()
    scale = (top / 127).float()
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double().unsqueeze(-1))
    return q, scale


def _plain_int8(x, wq, ws):
    if x.dtype == torch.bool:
        return (x.float() @ wq.t()) * ws                   # whole numbers below 2^24: exact in 32 bits
    q, scale = _plain_quantize(x)
    # sums of products up to 127^2: exact in 32 bits over 1024 terms, the parts added in 64
    total = torch.zeros(x.shape[0], wq.shape[0], dtype=torch.float64, device=x.device)
    for part in range(0, x.shape[1], 1024):
        total += (q[:, part:part + 1024].float() @ wq[:, part:part + 1024].t())
    return (total * scale.double().unsqueeze(-1) * ws.double()).to(x.dtype)


def _plain_delta(q, k, v, g, beta, initial, lengths):
    """The rule over chunks of 64 tokens: inside a chunk by products of triangular matrices, from chunk to chunk by the
    state."""
    t = v.dtype
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    n = -(-T // CHUNK)
    pad = n * CHUNK - T
    q, k, v, g, beta = q.float(), k.float(), v.float(), g.float(), beta.float()
    if lengths is not None:
        live = torch.arange(T, device=q.device) < lengths.unsqueeze(1)
        q, k, v = (torch.where(live[..., None, None], x, 0.0) for x in (q, k, v))
        g, beta = (torch.where(live[..., None], x, 0.0) for x in (g, beta))
    q, k = (x.repeat_interleave(Hv // Hk, 2) for x in (q, k))

    def chunks(x):                                          # (B, T, H, ...) -> (n, B, H, CHUNK, ...)
        x = torch.nn.functional.pad(x, [0, 0] * (x.dim() - 2) + [0, pad])
        x = x.reshape(B, n, CHUNK, *x.shape[2:]).transpose(2, 3)
        return x.transpose(0, 1)

    q, k, v, g, beta = chunks(q), chunks(k), chunks(v), chunks(g), chunks(beta).unsqueeze(-1)
    G = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    gamma = torch.exp(torch.where(low, (G.unsqueeze(-1) - G.unsqueeze(-2)).float(), -math.inf))
    A = beta * gamma * (k @ k.transpose(-1, -2)) * low.tril(-1)
    P = dk ** -0.5 * gamma * (q @ k.transpose(-1, -2))
    # the inverse of I + A by halves: blocks of 1, 2, 4, ... on the diagonal
    inv = torch.eye(CHUNK, device=q.device).expand_as(A)
    at = torch.arange(CHUNK, device=q.device)
    size = 1
    while size < CHUNK:
        corner = (at.unsqueeze(1) // size == at.unsqueeze(0) // size + 1) & (at.unsqueeze(1) // (2 * size) == at.unsqueeze(0) // (2 * size))
        inv = inv - inv @ (A * corner) @ inv
        size *= 2
    up = torch.exp(G.float()).unsqueeze(-1)
    down = torch.exp((G[..., -1:] - G).float()).unsqueeze(-1)
    last = torch.exp(G[..., -1].float())[..., None, None]
    S = initial.float() if initial is not None else torch.zeros(B, Hv, dk, dv, device=q.device)
    out = []
    for i in range(n):
        u = inv[i] @ (beta[i] * (v[i] - up[i] * (k[i] @ S)))
        out.append(dk ** -0.5 * up[i] * (q[i] @ S) + P[i] @ u)
        S = last[i] * S + (down[i] * k[i]).transpose(-1, -2) @ u
    o = torch.stack(out, 1).transpose(2, 3).reshape(B, n * CHUNK, Hv, dv)[:, :T]
    return o.to(t), S


def _plain_step(s):
    q, k, v = s['q'].float(), s['k'].float(), s['v'].float()
    group = v.shape[1] // k.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    S = s['initial']
    S *= torch.exp(s['g'])[..., None, None]
    u = s['beta'].unsqueeze(-1) * (v - (k.unsqueeze(-2) @ S).squeeze(-2))
    S += k.unsqueeze(-1) * u.unsqueeze(-2)
    o = q.shape[-1] ** -0.5 * (q.unsqueeze(-2) @ S).squeeze(-2)
    return o.to(s['v'].dtype), S


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def run(s):
    if s['op'] == 'int8':
        if own:
            from brainstate_b200 import EventArray
            return EventArray(s['x']) @ s['w8'] if s['x'].dtype == torch.bool else s['x'] @ s['w8']
        return _plain_int8(s['x'], s['wq'], s['ws'])
    if s['op'] == 'step':
        if own:
            from brainstate_b200 import plastic
            o = plastic.delta_rule_step(s['q'], s['k'], s['v'], s['g'], s['beta'], s['initial'])
            return {'o': o, 'state': s['initial']}
        o, state = _plain_step(s)
        return {'o': o, 'state': state}
    given = [s[n] for n in ('q', 'k', 'v', 'g', 'beta')]
    if own:
        from brainstate_b200 import plastic
        o, state = plastic.delta_rule(*given, initial_state=s['initial'], lengths=s['lengths'])
    else:
        o, state = _plain_delta(*given, s['initial'], s['lengths'])
    got = {'o': o, 'state': state}
    if s['op'] == 'train':
        leaves = [n for n in ('q', 'k', 'v', 'g', 'beta', 'initial') if s[n] is not None]
        grads = torch.autograd.grad((o, state), [s[n] for n in leaves], (s['do'], s['ds']))
        got.update({'d' + n: d for n, d in zip(leaves, grads)})
    return got


def work(case):
    size = {'float32': 4, 'bfloat16': 2, 'float16': 2, 'bool': 1}[case['dtype']]
    if case['op'] == 'int8':
        M, K, N = case['M'], case['K'], case['N']
        out = 4 if case['dtype'] == 'bool' else size
        return {'bytes': M * K * size + K * N + 4 * N + M * N * out, 'flops': 2 * M * K * N}
    B, T, Hk, Hv, dk, dv = (case[n] for n in ('B', 'T', 'Hk', 'Hv', 'dk', 'dv'))
    rows = B * T * ((2 * Hk * dk + Hv * dv) * size + 8 * Hv)      # q, k, v, g, beta
    outs = B * T * Hv * dv * size
    states = B * Hv * dk * dv * 4
    kept = states * (2 if case['state'] or case['op'] == 'step' else 1)
    flops = 6 * B * T * Hv * dk * dv                              # S^T k, k u^T and S^T q, each once
    if case['op'] == 'train':
        return {'bytes': 2 * rows + 2 * outs + 2 * kept, 'flops': 3 * flops}
    return {'bytes': rows + outs + kept, 'flops': flops}


# ---------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------

def _exact_int8(s):
    w = s['weight'].double()
    ws = (w.abs().max(0).values / 127).float().double()           # scales are 32-bit numbers by definition
    wq = (w / torch.where(ws == 0, 1.0, ws)).round()
    x = s['x'].double()
    if s['x'].dtype == torch.bool:
        return x @ wq * ws
    xs = (x.abs().max(1).values / 127).float().double()
    xq = (x / torch.where(xs == 0, 1.0, xs).unsqueeze(1)).round()
    return (xq @ wq) * ws * xs.unsqueeze(1)


def exact(case, seed):
    s = _make(case, seed)
    if case['op'] == 'int8':
        return _exact_int8(s)
    step = case['op'] == 'step'
    B, T, Hk, Hv, dk, dv = (case[n] for n in ('B', 'T', 'Hk', 'Hv', 'dk', 'dv'))
    train = case['op'] == 'train'
    if train and T * B * Hv * dk * dv * 8 > 40e9:
        return None
    q, k, v, g, beta = (s[n].double() for n in ('q', 'k', 'v', 'g', 'beta'))
    if step:
        q, k, v, g, beta = (x.unsqueeze(1) for x in (q, k, v, g, beta))
    live = torch.ones(B, T, 1, dtype=torch.float64, device=q.device)
    if s['lengths'] is not None:
        for b, n in enumerate(s['lengths'].tolist()):
            live[b, n:] = 0
    head = torch.arange(Hv, device=q.device) // (Hv // Hk)
    q, k = q[:, :, head], k[:, :, head]
    beta, a = beta * live, torch.exp(g * live)
    c = dk ** -0.5
    S = torch.zeros(B, Hv, dk, dv, dtype=torch.float64, device=q.device) if s['initial'] is None else s['initial'].double()
    o = torch.zeros_like(v)
    before, errs = [], []
    for t in range(T):                                             # token by token
        if train:
            before.append(S)
        aS = a[:, t, :, None, None] * S
        e = v[:, t] - torch.einsum('bhkv,bhk->bhv', aS, k[:, t])
        errs.append(e if train else None)
        S = aS + torch.einsum('bhk,bhv->bhkv', k[:, t], beta[:, t, :, None] * e)
        o[:, t] = c * live[:, t, :, None] * torch.einsum('bhkv,bhk->bhv', S, q[:, t])
    if step:
        return {'o': o[:, 0], 'state': S}
    got = {'o': o, 'state': S}
    if not train:
        return got
    do = s['do'].double() * live.unsqueeze(-1)
    dS = s['ds'].double()
    dq, dk_, dv_, dg, db = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    after = S
    for t in range(T - 1, -1, -1):
        S0, e, kt, bt, at = before[t], errs[t], k[:, t], beta[:, t, :, None], a[:, t, :, None]
        dS = dS + c * torch.einsum('bhk,bhv->bhkv', q[:, t], do[:, t])
        dq[:, t] = c * torch.einsum('bhkv,bhv->bhk', after, do[:, t])
        du = torch.einsum('bhkv,bhk->bhv', dS, kt)
        db[:, t] = (du * e).sum(-1) * live[:, t]
        dv_[:, t] = bt * du
        dk_[:, t] = torch.einsum('bhkv,bhv->bhk', dS, bt * e) - at * torch.einsum('bhkv,bhv->bhk', S0, bt * du)
        dS = dS - torch.einsum('bhk,bhv->bhkv', kt, bt * du)
        dg[:, t] = at[..., 0] * (dS * S0).sum((-1, -2)) * live[:, t]
        dS = at.unsqueeze(-1) * dS
        after = S0
    dk_ = dk_ * live.unsqueeze(-1)
    got['dq'] = dq.reshape(B, T, Hk, Hv // Hk, dk).sum(3)
    got['dk'] = dk_.reshape(B, T, Hk, Hv // Hk, dk).sum(3)
    got['dv'], got['dg'], got['dbeta'] = dv_, dg, db
    if s['initial'] is not None:
        got['dinitial'] = dS
    return got
