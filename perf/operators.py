"""The sequence-layer operators this framework is timed on, and their plain forms.

A layer that carries fast weights from token to token: a key/value state trained and prefilled in
chunks and advanced token by token when it answers (``delta``, ``delta_train``, ``delta_step``),
the norms, gate and residual around it (``norm``, ``norm_train``), and its projections in 8-bit
integers when it serves (``int8``).

With q, k [.., dk], v [.., dv], log decay g <= 0 and write strength beta of one head and token:

    S'_t = exp(g_t) S_{t-1}                     (S [dk, dv])
    u_t  = beta_t (v_t - S'_t^T k_t)
    S_t  = S'_t + k_t u_t^T
    o_t  = scale S_t^T q_t                      (scale = dk^-1/2)

The norms around a block's output y, with r(x) = x / sqrt(mean(x^2) + eps):

    stream = residual + scale * silu(gate) * (r(y) * post_weight),  normed = r(stream) * pre_weight

The integer product, for tokens x and weights w8 with a scale for each output channel:

    a = max|x| / 127,  x8 = round(x / a),  y = a * w_scale * (x8 . w8) + bias
"""
import torch

own = False

_DEV = 'cuda'
_TYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
_EPS = 1e-6


def listed():
    return [
        # a long prompt through a wide layer: keys shared by two value heads each
        dict(name='delta_prefill_8k', kind='delta', batch=1, tokens=8192, seqs=0, hk=16, hv=32,
             dk=128, dv=128, dtype='bf16'),
        # prompts of many lengths packed end to end, an empty one and single tokens among them
        dict(name='delta_prefill_ragged', kind='delta', batch=1, tokens=5003, seqs=13, hk=4, hv=8,
             dk=64, dv=80, dtype='f16'),
        # one training step's layer, forward and backward
        dict(name='delta_train_2k', kind='delta_train', batch=4, tokens=2048, seqs=0, hk=8, hv=16,
             dk=128, dv=128, dtype='bf16'),
        # a small odd layer trained in 32 bits on short sequences
        dict(name='delta_train_odd', kind='delta_train', batch=2, tokens=333, seqs=0, hk=3, hv=3,
             dk=48, dv=72, dtype='f32'),
        # one user's next token: latency
        dict(name='delta_step_1', kind='delta_step', batch=1, slots=4, hk=16, hv=32, dk=128,
             dv=128, dtype='bf16'),
        # a full serving batch, some of its rows idle: the states' bytes
        dict(name='delta_step_256', kind='delta_step', batch=256, slots=320, hk=16, hv=32, dk=128,
             dv=128, dtype='bf16'),
        # between two blocks when one token is answered: latency
        dict(name='norm_step', kind='norm', rows=2, dim=4096, post=True, gate=True, scale=True,
             residual=True, pre=True, dtype='bf16'),
        # the same over a long prompt
        dict(name='norm_prefill', kind='norm', rows=8192, dim=4096, post=True, gate=True,
             scale=True, residual=True, pre=True, dtype='bf16'),
        # and in training, at odd sizes
        dict(name='norm_train_odd', kind='norm_train', rows=4099, dim=2050, post=True, gate=True,
             scale=True, residual=True, pre=True, dtype='bf16'),
        # a projection of one token: the weight's bytes
        dict(name='int8_step', kind='int8', tokens=1, n_in=4096, n_out=4096, bias=False,
             dtype='bf16'),
        # a small ragged layer
        dict(name='int8_ragged', kind='int8', tokens=77, n_in=1000, n_out=300, bias=True,
             dtype='f32'),
        # a projection of a long prompt
        dict(name='int8_prefill', kind='int8', tokens=8192, n_in=4096, n_out=4096, bias=True,
             dtype='bf16'),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; round numbers and odd ones."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.4:
        v = max(lo, v // 16 * 16)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(['delta', 'delta', 'delta_train', 'delta_train', 'delta_step', 'norm',
                       'norm', 'norm_train', 'int8', 'int8'])
    dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    if kind.startswith('delta'):
        hk = rng.choice([1, 2, 3, 4, 8, 16])
        c = dict(kind=kind, batch=1, hk=hk, hv=hk * rng.choice([1, 1, 2, 4]),
                 dk=rng.choice([128, 128, 64, 96, rng.randint(16, 128)]),
                 dv=rng.choice([128, 128, 64, 80, rng.randint(16, 128)]), dtype=dtype)
        c['hv'] = min(c['hv'], 32 // hk * hk)
        per_token = c['hv'] * c['dk'] * c['dv']
        if kind == 'delta_step':
            c['batch'] = min(_log(rng, 1, 256), 256 * 32 * 16384 // per_token)
            c['slots'] = c['batch'] + rng.randint(0, 64)
            return c
        most = (8192 * 32 if kind == 'delta' else 8192 * 16) * 16384 // per_token
        c['tokens'] = min(_log(rng, 1, 8192) if kind == 'delta' else _log(rng, 8, 4096), most)
        c['seqs'] = _log(rng, 2, 40) if rng.random() < 0.4 else 0
        if not c['seqs']:
            c['batch'] = min(_log(rng, 1, 16), max(1, most // c['tokens']))
        return c
    if kind.startswith('norm'):
        dim = _log(rng, 64, 8192)
        c = dict(kind=kind, rows=min(_log(rng, 1, 32768), 8192 * 4096 // dim), dim=dim)
        if kind == 'norm_train':
            c['rows'] = min(c['rows'], 4099 * 2050 // dim)
        form = rng.choice(['all', 'all', 'head', 'plain', 'pre'])
        # everything; a head's norm and gate; residual and norm; the norm alone
        c.update(post=form in ('all', 'head'), gate=form in ('all', 'head'), scale=form == 'all',
                 residual=form in ('all', 'plain'), pre=form in ('all', 'plain', 'pre'),
                 dtype=dtype)
        return c
    n_in, n_out = _log(rng, 64, 8192), _log(rng, 64, 8192)
    return dict(kind='int8', tokens=min(_log(rng, 1, 8192), 8192 * 4096 * 4096 // (n_in * n_out)),
                n_in=n_in, n_out=n_out, bias=rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """Lengths of the packed sequences: an empty one, single tokens, the others uneven."""
    n, total = case['seqs'], case['tokens']
    w = [(7 * i * i + 3 * i) % 11 + 1 for i in range(n)]
    w[1 % n] = 0
    cuts, at = [0], 0
    for i in range(n):
        at += w[i]
        cuts.append(total * at // sum(w))
    lens = [b - a for a, b in zip(cuts, cuts[1:])]
    if n > 3 and lens[0] > 1:
        lens[2], lens[0] = lens[2] + lens[0] - 1, 1
    return lens


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    dtype = _TYPES[case['dtype']]

    def randn(*shape, sd=1.0):
        return torch.randn(shape, generator=gen, device=_DEV) * sd

    s = dict(case=case, kind=case['kind'])
    if s['kind'].startswith('delta'):
        b, hk, hv, dk, dv = (case[n] for n in ('batch', 'hk', 'hv', 'dk', 'dv'))
        lead = (b,) if s['kind'] == 'delta_step' else (b, case['tokens'])
        q, k = (torch.nn.functional.silu(randn(*lead, hk, dk)) for _ in range(2))
        s['q'], s['k'] = ((x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)).to(dtype)
                          for x in (q, k))
        s['v'] = torch.nn.functional.silu(randn(*lead, hv, dv)).to(dtype)
        # decays of a head from slow to fast, write strengths in (0, 1)
        rate = torch.linspace(0.02, 2.0, hv, device=_DEV)
        s['g'] = -rate * torch.nn.functional.softplus(randn(*lead, hv) - 2)
        s['beta'] = torch.sigmoid(randn(*lead, hv)).to(dtype)
        if s['kind'] == 'delta_step':
            s['state'] = randn(case['slots'], hv, dk, dv, sd=0.1)
            slots = torch.randperm(case['slots'], generator=gen, device=_DEV)[:b].to(torch.int32)
            if b > 8:
                slots[::8] = -1                      # idle rows
            s['slots'] = slots
            return s
        s['offsets'], s['max_len'], n = None, case['tokens'], b
        if case['seqs']:
            lens = _lengths(case)
            s['offsets'] = torch.tensor([0] + lens, device=_DEV).cumsum(0).to(torch.int32)
            s['max_len'], n = max(lens), len(lens)
        if s['kind'] == 'delta':
            s['state'] = randn(n, hv, dk, dv, sd=0.1)
        else:
            s['do'] = randn(*lead, hv, dv, sd=0.1).to(dtype)
        return s
    if s['kind'].startswith('norm'):
        rows, dim = case['rows'], case['dim']
        s['y'] = (randn(rows, dim) * (0.5 + torch.rand(rows, 1, generator=gen, device=_DEV))
                  ).to(dtype)
        s['post'] = (1 + randn(dim, sd=0.1)) if case['post'] else None
        s['gate'] = randn(rows, dim).to(dtype) if case['gate'] else None
        s['scale'] = (0.5 + randn(dim, sd=0.1)) if case['scale'] else None
        s['residual'] = randn(rows, dim, sd=2.0).to(dtype) if case['residual'] else None
        s['pre'] = (1 + randn(dim, sd=0.1)) if case['pre'] else None
        if s['kind'] == 'norm_train':
            s['dstream'] = randn(rows, dim, sd=0.1).to(dtype)
            s['dnormed'] = randn(rows, dim, sd=0.1).to(dtype) if case['pre'] else None
        return s
    t, n_in, n_out = case['tokens'], case['n_in'], case['n_out']
    s['x'] = (randn(t, n_in) * (0.2 + torch.rand(t, 1, generator=gen, device=_DEV))).to(dtype)
    s['w8'] = randn(n_out, n_in, sd=32.0).round().clamp(-127, 127).to(torch.int8)
    s['w_scale'] = (0.5 + torch.rand(n_out, generator=gen, device=_DEV)) * 0.02 / n_in ** 0.5
    s['bias'] = randn(n_out, sd=0.1).to(dtype) if case['bias'] else None
    return s


# ------------------------------------------------------------------------------ plain forms
_CHUNK = 64


def _plain_delta(q, k, v, g, beta, state, offsets=None, max_len=None):
    """The recurrence over chunks of 64 tokens in 32 bits; sequences packed end to end are laid
    side by side first (tokens past a sequence's end have no decay and write nothing)."""
    kind = v.dtype
    q, k, v, g, beta = (x.float() for x in (q, k, v, g, beta))
    if offsets is not None:
        at = offsets[:-1, None].long() + torch.arange(max_len, device=_DEV)
        inside = at < offsets[1:, None]
        at = at.clamp(max=q.shape[1] - 1)
        q, k, v, g, beta = (x[0][at] * inside.reshape(inside.shape + (1,) * (x.dim() - 2))
                            for x in (q, k, v, g, beta))
    b, t, hv, dv = v.shape
    dk, group, n = q.shape[-1], hv // q.shape[2], -(-t // _CHUNK)

    def chunks(x, rep=1):
        x = x.unsqueeze(-1) if x.dim() == 3 else x
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * _CHUNK - t))
        x = x.permute(0, 2, 1, 3).reshape(b, x.shape[2], n, _CHUNK, x.shape[3])
        return x.repeat_interleave(rep, 1) if rep > 1 else x

    q, k, v = chunks(q, group) * dk ** -0.5, chunks(k, group), chunks(v)
    beta, run_g = chunks(beta), chunks(g).cumsum(3)
    i = torch.arange(_CHUNK, device=_DEV)
    diff = run_g - run_g.transpose(3, 4)
    decay = torch.where(i[:, None] >= i, diff, torch.full_like(diff, -1e30)).exp()
    power = -(beta * decay * (k @ k.transpose(3, 4))) * (i[:, None] > i)
    inv = torch.eye(_CHUNK, device=_DEV) + power       # (1 - power)^-1 by its doubling product
    for _ in range(5):
        power = power @ power
        inv = inv + inv @ power
    att = decay * (q @ k.transpose(3, 4))
    grow = run_g.exp()
    left = (run_g[:, :, :, -1:] - run_g).exp()
    out = []
    for c in range(n):
        u = inv[:, :, c] @ (beta[:, :, c] * (v[:, :, c] - (grow[:, :, c] * k[:, :, c]) @ state))
        out.append((grow[:, :, c] * q[:, :, c]) @ state + att[:, :, c] @ u)
        state = grow[:, :, c, -1:] * state + (left[:, :, c] * k[:, :, c]).transpose(2, 3) @ u
    o = torch.stack(out, 2).reshape(b, hv, n * _CHUNK, dv)[:, :, :t].transpose(1, 2)
    if offsets is not None:
        o = o[inside].unsqueeze(0)
    return o.to(kind), state


def _plain_delta_step(q, k, v, g, beta, state, slots):
    kind, group = v.dtype, v.shape[1] // q.shape[1]
    q, k, v, g, beta = (x.float() for x in (q, k, v, g, beta))
    q, k = (x.repeat_interleave(group, 1) if group > 1 else x for x in (q, k))
    live = slots >= 0
    at = slots.clamp(min=0).long()
    s = state[at] * g.exp()[:, :, None, None]
    u = beta[..., None] * (v - (s * k[..., None]).sum(2))
    s = s + k[..., None] * u[:, :, None]
    o = (s * q[..., None]).sum(2) * q.shape[-1] ** -0.5
    state[at[live]] = s[live]
    return (o * live[:, None, None]).to(kind)


def _plain_norm(y, post, gate, scale, residual, pre):
    kind = y.dtype
    t = y.float()
    if post is not None:
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + _EPS) * post.float()
    if gate is not None:
        z = gate.float()
        t = t * (z / (1 + (-z).exp()))
    if scale is not None:
        t = t * scale.float()
    if residual is not None:
        t = t + residual.float()
    if pre is None:
        return t.to(kind), None
    return t.to(kind), (t * torch.rsqrt((t * t).mean(-1, keepdim=True) + _EPS)
                        * pre.float()).to(kind)


def _plain_int8(x, w8, w_scale, bias):
    f = x.float()
    a = f.abs().amax(-1, keepdim=True) / 127
    x8 = torch.where(a > 0, (f / a).round(), torch.zeros_like(f))
    y = (x8 @ w8.float().t()) * (a * w_scale)
    return (y + bias.float() if bias is not None else y).to(x.dtype)


# ------------------------------------------------------------------------------ one pass
def run(s):
    kind = s['kind']
    if own:
        from brainstate_amd import ops
    if kind == 'delta':
        if own:
            return ops.gated_delta_rule(s['q'], s['k'], s['v'], s['g'], s['beta'],
                                        initial_state=s['state'], seq_offsets=s['offsets'])
        return _plain_delta(s['q'], s['k'], s['v'], s['g'], s['beta'], s['state'], s['offsets'],
                            s['max_len'])
    if kind == 'delta_train':
        args = [s[n].detach().requires_grad_() for n in ('q', 'k', 'v', 'g', 'beta')]
        with torch.enable_grad():
            if own:
                o = ops.gated_delta_rule(*args, seq_offsets=s['offsets'])[0]
            else:
                n = s['offsets'].numel() - 1 if s['offsets'] is not None else s['q'].shape[0]
                zero = torch.zeros(n, s['v'].shape[2], s['q'].shape[3], s['v'].shape[3],
                                   device=_DEV)
                o = _plain_delta(*args, zero, s['offsets'], s['max_len'])[0]
        return (o.detach(),) + torch.autograd.grad(o, args, s['do'])
    if kind == 'delta_step':
        step = ops.gated_delta_step if own else _plain_delta_step
        o = step(s['q'], s['k'], s['v'], s['g'], s['beta'], s['state'], slots=s['slots'])
        return o, s['state']
    if kind == 'norm':
        args = (s['y'], s['post'], s['gate'], s['scale'], s['residual'], s['pre'])
        if own:
            return ops.norm_gate_residual(s['y'], post_weight=s['post'], gate=s['gate'],
                                          scale=s['scale'], residual=s['residual'],
                                          pre_weight=s['pre'], eps=_EPS)
        return _plain_norm(*args)
    if kind == 'norm_train':
        args = {n: s[n].detach().requires_grad_() for n in
                ('y', 'post', 'gate', 'scale', 'residual', 'pre') if s[n] is not None}
        with torch.enable_grad():
            a = [args.get(n) for n in ('y', 'post', 'gate', 'scale', 'residual', 'pre')]
            if own:
                outs = ops.norm_gate_residual(a[0], post_weight=a[1], gate=a[2], scale=a[3],
                                              residual=a[4], pre_weight=a[5], eps=_EPS)
            else:
                outs = _plain_norm(*a)
        pairs = [(o, d) for o, d in zip(outs, (s['dstream'], s['dnormed'])) if o is not None]
        grads = torch.autograd.grad([o for o, _ in pairs], list(args.values()),
                                    [d for _, d in pairs])
        return tuple(o.detach() for o, _ in pairs) + grads
    if own:
        return ops.int8_linear(s['x'], s['w8'], s['w_scale'], bias=s['bias'])
    return _plain_int8(s['x'], s['w8'], s['w_scale'], s['bias'])


def work(case):
    kind, size = case['kind'], 4 if case['dtype'] == 'f32' else 2
    if kind.startswith('delta'):
        hk, hv, dk, dv, b = (case[n] for n in ('hk', 'hv', 'dk', 'dv', 'batch'))
        n = b * (1 if kind == 'delta_step' else case['tokens'])
        qk, vo, gate = 2 * n * hk * dk * size, 2 * n * hv * dv * size, n * hv * (4 + size)
        cell = n * hv * dk * dv
        if kind == 'delta_step':
            live = b - len(range(0, b, 8)) if b > 8 else b
            return dict(bytes=qk + vo + gate + 8 * live * hv * dk * dv, flops=8 * cell * live // b)
        # state read, written and queried (3 products of dk x dv a token), and the products
        # within a chunk of 64
        flops = 6 * cell + n * hv * 64 * 2 * (2 * dk + 2 * dv)
        if kind == 'delta':
            n_seq = case['seqs'] or b
            return dict(bytes=qk + vo + gate + 8 * n_seq * hv * dk * dv, flops=flops)
        # backward: q, k, v, g, beta and the output's gradient in, five gradients out
        return dict(bytes=qk + vo + gate + 2 * qk + vo + vo // 2 + 2 * gate, flops=3 * flops)
    if kind.startswith('norm'):
        n, d = case['rows'] * case['dim'], case['dim']
        ins = 1 + case['gate'] + case['residual']
        outs = 1 + case['pre']
        w = 4 * d * (case['post'] + case['scale'] + case['pre'])
        if kind == 'norm':
            return dict(bytes=n * size * (ins + outs) + w, flops=12 * n)
        return dict(bytes=n * size * (ins + outs) + w + n * size * (2 * ins + outs) + 2 * w,
                    flops=40 * n)
    t, n_in, n_out = case['tokens'], case['n_in'], case['n_out']
    return dict(bytes=t * n_in * size + n_in * n_out + 4 * n_out + t * n_out * size,
                flops=2 * t * n_in * n_out)


# ------------------------------------------------------------------------------ in 64 bits
def _exact_delta(q, k, v, g, beta, state, do=None):
    """Token by token in 64 bits, [B, T, H, d] with as many key heads as value heads; with
    ``do`` the gradients too, by the recurrence's own transpose."""
    t, scale = q.shape[1], q.shape[-1] ** -0.5
    o = torch.empty_like(v)
    kept = []
    for i in range(t):
        if do is not None:
            kept.append(state)
        ki, decay = k[:, i, :, :, None], g[:, i].exp()[..., None, None]
        s = decay * state
        u = beta[:, i, :, None] * (v[:, i] - (s * ki).sum(2))
        state = s + ki * u[:, :, None]
        o[:, i] = scale * (state * q[:, i, :, :, None]).sum(2)
    if do is None:
        return o, state
    ds = torch.zeros_like(state)
    dq, dk, dv, dg, db = (torch.empty_like(x) for x in (q, k, v, g, beta))
    for i in reversed(range(t)):
        ki, qi, doi = k[:, i, :, :, None], q[:, i, :, :, None], do[:, i, :, None]
        decay = g[:, i].exp()[..., None, None]
        s = decay * kept[i]
        miss = v[:, i] - (s * ki).sum(2)
        u = beta[:, i, :, None] * miss
        dq[:, i] = scale * ((s + ki * u[:, :, None]) * doi).sum(3)
        ds = ds + scale * qi * doi
        du = (ds * ki).sum(2)
        dmiss = beta[:, i, :, None] * du
        db[:, i] = (du * miss).sum(2)
        dv[:, i] = dmiss
        dk[:, i] = (ds * u[:, :, None]).sum(3) - (s * dmiss[:, :, None]).sum(3)
        ds = ds - ki * dmiss[:, :, None]
        dg[:, i] = (ds * s).sum((2, 3))
        ds = decay * ds
    return o, dq, dk, dv, dg, db


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind.startswith('delta'):
        hk, group = case['hk'], case['hv'] // case['hk']
        x = [s[n].double() for n in ('q', 'k', 'v', 'g', 'beta')]
        x[:2] = [a.repeat_interleave(group, -2) for a in x[:2]]
        if kind == 'delta_step':
            x = [a.unsqueeze(1) for a in x]
            state, live = s['state'].double(), s['slots'] >= 0
            at = s['slots'][live].long()
            o = torch.zeros_like(x[2])
            o[live], state[at] = _exact_delta(*(a[live] for a in x), state[at])
            return o[:, 0], state
        if s['offsets'] is not None:
            lens = _lengths(case)

            def side_by_side(a):
                parts = a[0].split(lens)
                p = torch.zeros((len(lens), max(lens)) + a.shape[2:], dtype=a.dtype, device=_DEV)
                for i, part in enumerate(parts):
                    p[i, :lens[i]] = part
                return p

            def packed(a):
                return torch.cat([a[i, :n] for i, n in enumerate(lens)]).unsqueeze(0)
        else:
            side_by_side = packed = lambda a: a                              # noqa: E731
        x = [side_by_side(a) for a in x]
        if kind == 'delta':
            o, state = _exact_delta(*x, s['state'].double())
            return packed(o), state
        zero = torch.zeros(x[0].shape[0], case['hv'], case['dk'], case['dv'], device=_DEV,
                           dtype=torch.float64)
        if zero.numel() * 8 * x[0].shape[1] > 60e9:
            return None
        r = [packed(a) for a in _exact_delta(*x, zero, side_by_side(s['do'].double()))]
        r[1:3] = [a.reshape(a.shape[:2] + (hk, group, a.shape[3])).sum(3) for a in r[1:3]]
        return tuple(r)
    if kind.startswith('norm'):
        x = {n: s[n].double() if s[n] is not None else None
             for n in ('y', 'post', 'gate', 'scale', 'residual', 'pre')}
        y = x['y']
        r1 = (y.square().mean(1, keepdim=True) + _EPS) ** -0.5 if case['post'] else 1.0
        w1 = x['post'] if case['post'] else 1.0
        sg = torch.sigmoid(x['gate']) if case['gate'] else 1.0
        act = x['gate'] * sg if case['gate'] else 1.0
        c = x['scale'] if case['scale'] else 1.0
        stream = y * r1 * w1 * act * c + (x['residual'] if case['residual'] else 0.0)
        outs = [stream]
        if case['pre']:
            r2 = (stream.square().mean(1, keepdim=True) + _EPS) ** -0.5
            outs.append(stream * r2 * x['pre'])
        if kind == 'norm':
            return tuple(outs) if case['pre'] else (stream, None)
        d = s['dstream'].double()
        dpre = None
        if case['pre']:
            n, dn = stream * r2, s['dnormed'].double()
            dpre = (dn * n).sum(0)
            dn = dn * x['pre']
            d = d + r2 * (dn - n * (dn * n).mean(1, keepdim=True))
        grads = {'residual': d, 'pre': dpre, 'scale': (d * y * r1 * w1 * act).sum(0)}
        if case['gate']:
            grads['gate'] = d * c * y * r1 * w1 * sg * (1 + x['gate'] * (1 - sg))
        dp = d * c * act
        dy = dp
        if case['post']:
            n = y * r1
            grads['post'] = (dp * n).sum(0)
            dp = dp * w1
            dy = r1 * (dp - n * (dp * n).mean(1, keepdim=True))
        grads['y'] = dy
        return tuple(outs) + tuple(grads[n] for n in x if x[n] is not None)
    f = s['x'].double()
    a = f.abs().amax(1, keepdim=True) / 127
    x8 = torch.where(a > 0, torch.round(f / a), torch.zeros_like(f))
    y = (x8 @ s['w8'].double().t()) * a * s['w_scale'].double()
    return y + s['bias'].double() if case['bias'] else y
