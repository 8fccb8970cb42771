"""More sequence-layer operators this framework is timed on, and their plain forms.

A layer whose memory fades at a rate of its own for each head, trained and prefilled in chunks
(``decay``, ``decay_train``) and advanced token by token when it answers (``decay_step``); layer
norm, alone when it answers (``norm``) and trained behind a dropped-out branch and its residual
(``norm_train``); dropout whose mask is never stored (``dropout``); and projections with 4-bit
weights when it serves (``int4``).

With q, k [.., dk], v [.., dv] and log decay g <= 0 of one head and token:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T          (S [dk, dv])
    o_t = scale S_t^T q_t                       (scale = dk^-1/2)

g has a value for each token and head, or one for each head.  Dropout of the element in row r and
column c keeps it, times 1 / (1 - p), where word c % 4 of the Philox 4x32-10 generator (Salmon et
al. 2011) with counter (c / 4, site, r mod 2^32, r / 2^32) and the seed's two halves as its key is at
least p 2^32.  Layer norm and its gradients, over rows of n:

    stream = residual + dropout(x),  h = (stream - mean) / sqrt(var + eps),  normed = h weight + bias

4-bit weights u in 0..15 [n_out, n_in] lie two to a byte, the even one in the low half, with a scale
for each channel and group of input values:

    y_mn = sum_k x_mk (u_nk - 8) scale_n,k/group + bias_n
"""
import numpy as np
import torch

own = False

_DEV = 'cuda'
_TYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
_EPS = 1e-5


def listed():
    return [
        # a long prompt through a wide layer whose tokens each have their own decay
        dict(name='decay_prefill_8k', kind='decay', batch=1, tokens=8192, seqs=0, hk=32, hv=32,
             dk=128, dv=128, each=True, dtype='bf16'),
        # prompts of many lengths packed end to end, an empty one and single tokens among them;
        # keys shared by two value heads each, one decay a head
        dict(name='decay_prefill_ragged', kind='decay', batch=1, tokens=5003, seqs=13, hk=4, hv=8,
             dk=64, dv=80, each=False, dtype='f16'),
        # one training step's layer, forward and backward
        dict(name='decay_train_2k', kind='decay_train', batch=4, tokens=2048, seqs=0, hk=16,
             hv=16, dk=128, dv=128, each=True, dtype='bf16'),
        # a small odd layer trained in 32 bits on short sequences
        dict(name='decay_train_odd', kind='decay_train', batch=2, tokens=333, seqs=0, hk=3, hv=3,
             dk=48, dv=72, each=False, dtype='f32'),
        # one user's next token: latency
        dict(name='decay_step_1', kind='decay_step', batch=1, slots=4, hk=32, hv=32, dk=128,
             dv=128, each=True, dtype='bf16'),
        # a full serving batch, some of its rows idle: the states' bytes
        dict(name='decay_step_256', kind='decay_step', batch=256, slots=320, hk=32, hv=32, dk=128,
             dv=128, each=False, dtype='bf16'),
        # a block's norm when one token of two rows is answered: latency
        dict(name='layer_norm_step', kind='norm', rows=2, dim=4096, dtype='bf16'),
        # a block's dropped-out branch, residual and norm in a training step
        dict(name='layer_norm_train', kind='norm_train', rows=8192, dim=4096, p=0.1, dtype='bf16'),
        # dropout of a wide activation in a training step, forward and backward
        dict(name='dropout_train', kind='dropout', rows=8192, dim=4096, p=0.1, dtype='bf16'),
        # and of a small odd one
        dict(name='dropout_odd', kind='dropout', rows=333, dim=217, p=0.5, dtype='f32'),
        # a projection of one token: the weight's bytes
        dict(name='int4_step', kind='int4', tokens=1, n_in=4096, n_out=4096, group=128,
             bias=False, dtype='bf16'),
        # a projection of a long prompt
        dict(name='int4_prefill', kind='int4', tokens=8192, n_in=4096, n_out=4096, group=128,
             bias=True, dtype='bf16'),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; round numbers and odd ones."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.4:
        v = max(lo, v // 16 * 16)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(['decay', 'decay', 'decay_train', 'decay_train', 'decay_step', 'norm',
                       'norm_train', 'norm_train', 'dropout', 'int4', 'int4', 'int4'])
    dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    if kind.startswith('decay'):
        hk = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = dict(kind=kind, batch=1, hk=hk, hv=min(hk * rng.choice([1, 1, 2, 4]), 32 // hk * hk),
                 dk=rng.choice([128, 128, 64, 96, rng.randint(16, 128)]),
                 dv=rng.choice([128, 128, 64, 80, rng.randint(16, 128)]),
                 each=rng.random() < 0.5, dtype=dtype)
        per_token = c['hv'] * c['dk'] * c['dv']
        if kind == 'decay_step':
            c['batch'] = min(_log(rng, 1, 256), 256 * 32 * 16384 // per_token)
            c['slots'] = c['batch'] + rng.randint(0, 64)
            return c
        most = (8192 * 32 if kind == 'decay' else 8192 * 16) * 16384 // per_token
        c['tokens'] = min(_log(rng, 1, 8192) if kind == 'decay' else _log(rng, 8, 4096), most)
        c['seqs'] = _log(rng, 2, 40) if rng.random() < 0.4 else 0
        if not c['seqs']:
            c['batch'] = min(_log(rng, 1, 16), max(1, most // c['tokens']))
        return c
    if kind == 'int4':
        n_in, n_out = _log(rng, 64, 8192), _log(rng, 64, 8192)
        return dict(kind=kind, n_in=n_in, n_out=n_out, group=rng.choice([128, 128, 64, 32]),
                    tokens=min(rng.choice([1, _log(rng, 1, 16), _log(rng, 1, 8192)]),
                               8192 * 4096 * 4096 // (n_in * n_out)),
                    bias=rng.random() < 0.5, dtype=dtype)
    dim = _log(rng, 64, 8192)
    c = dict(kind=kind, rows=min(_log(rng, 1, 32768), 8192 * 4096 // dim), dim=dim, dtype=dtype)
    if kind == 'norm_train':
        c['p'] = rng.choice([0.0, 0.1, 0.1, 0.3])
    if kind == 'dropout':
        c['p'] = rng.choice([0.1, 0.1, 0.25, 0.5])
    return c


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
    if s['kind'].startswith('decay'):
        b, hk, hv, dk, dv = (case[n] for n in ('batch', 'hk', 'hv', 'dk', 'dv'))
        lead = (b,) if s['kind'] == 'decay_step' else (b, case['tokens'])
        q, k = (torch.nn.functional.silu(randn(*lead, hk, dk)) for _ in range(2))
        s['q'], s['k'] = ((x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)).to(dtype)
                          for x in (q, k))
        s['v'] = torch.nn.functional.silu(randn(*lead, hv, dv)).to(dtype)
        # decays of a head from slow to fast
        rate = torch.logspace(-2.5, 0, hv, device=_DEV)
        s['g'] = -rate * (torch.nn.functional.softplus(randn(*lead, hv)) if case['each'] else
                          0.5 + torch.rand(hv, generator=gen, device=_DEV))
        if s['kind'] == 'decay_step':
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
        if s['kind'] == 'decay':
            s['state'] = randn(n, hv, dk, dv, sd=0.1)
        else:
            s['do'] = randn(*lead, hv, dv, sd=0.1).to(dtype)
        return s
    if s['kind'] == 'int4':
        t, n_in, n_out, group = (case[n] for n in ('tokens', 'n_in', 'n_out', 'group'))
        s['x'] = (randn(t, n_in) * (0.2 + torch.rand(t, 1, generator=gen, device=_DEV))).to(dtype)
        u = (8 + randn(n_out, n_in + n_in % 2, sd=2.6)).round().clamp(1, 15).to(torch.uint8)
        s['w4'] = u[:, ::2] | u[:, 1::2] << 4
        s['w_scale'] = (0.5 + torch.rand(n_out, -(-n_in // group), generator=gen, device=_DEV)
                        ) * 0.3 / n_in ** 0.5
        s['bias'] = randn(n_out, sd=0.1).to(dtype) if case['bias'] else None
        return s
    rows, dim = case['rows'], case['dim']
    s['x'] = (randn(rows, dim) * (0.5 + torch.rand(rows, 1, generator=gen, device=_DEV))
              + randn(rows, 1, sd=0.3)).to(dtype)
    s['seed'], s['site'] = (seed * 0x9E3779B97F4A7C15 + 1) % 2 ** 63, 5
    if s['kind'] == 'dropout':
        s['dy'] = randn(rows, dim, sd=0.1).to(dtype)
        return s
    s['weight'], s['bias'] = 1 + randn(dim, sd=0.1), randn(dim, sd=0.1)
    if s['kind'] == 'norm_train':
        s['residual'] = randn(rows, dim, sd=2.0).to(dtype)
        s['dstream'], s['dnormed'] = (randn(rows, dim, sd=0.1).to(dtype) for _ in range(2))
    return s


# ------------------------------------------------------------------------------ plain forms
_CHUNK = 64


def _plain_decay(q, k, v, g, state, offsets=None, max_len=None):
    """Chunks of 64 tokens, all at once: what each leaves in the state, the states between them by
    the decays from chunk to chunk, and what each reads.  Products in 32 bits, decays' sums in 64;
    sequences packed end to end are laid side by side first (tokens past a sequence's end have no
    decay and write nothing)."""
    kind = v.dtype
    q, k, v = (x.float() for x in (q, k, v))
    g = g.double().expand(v.shape[:3])
    if offsets is not None:
        at = offsets[:-1, None].long() + torch.arange(max_len, device=_DEV)
        inside = at < offsets[1:, None]
        at = at.clamp(max=q.shape[1] - 1)
        q, k, v, g = (x[0][at] * inside.reshape(inside.shape + (1,) * (x.dim() - 2))
                      for x in (q, k, v, g))
    b, t, hv, dv = v.shape
    dk, group, n = q.shape[-1], hv // q.shape[2], -(-t // _CHUNK)

    def chunks(x, rep=1):
        x = x.unsqueeze(-1) if x.dim() == 3 else x
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * _CHUNK - t))
        x = x.permute(0, 2, 1, 3).reshape(b, x.shape[2], n, _CHUNK, x.shape[3])
        return x.repeat_interleave(rep, 1) if rep > 1 else x

    q, k, v = chunks(q, group) * dk ** -0.5, chunks(k, group), chunks(v)
    run = chunks(g).cumsum(3)                           # within a chunk
    total = run[:, :, :, -1, 0].cumsum(2)               # up to a chunk's end
    i = torch.arange(_CHUNK, device=_DEV)
    diff = run - run.transpose(3, 4)
    att = torch.where(i[:, None] >= i, diff, torch.full_like(diff, -1e30)).exp().float() * (
        q @ k.transpose(3, 4))
    left = (run[:, :, :, -1:] - run).exp().float()
    adds = (left * k).transpose(3, 4) @ v               # [b, hv, n, dk, dv]
    # before chunk c there is what chunk x < c added, decayed over the chunks between them
    before = torch.cat([torch.zeros_like(total[:, :, :1]), total[:, :, :-1]], 2)
    j = torch.arange(n, device=_DEV)
    diff = torch.cat([before, total[:, :, -1:]], 2)[:, :, :, None] - total[:, :, None]
    mix = torch.where(torch.arange(n + 1, device=_DEV)[:, None] > j, diff,
                      torch.full_like(diff, -1e30)).exp().float()
    states = (mix @ adds.reshape(b, hv, n, dk * dv)).reshape(b, hv, n + 1, dk, dv)
    if state is not None:
        grow = torch.cat([before, total[:, :, -1:]], 2).exp().float()
        states = states + grow[..., None, None] * state[:, :, None]
    o = (run.exp().float() * q) @ states[:, :, :-1] + att @ v
    o = o.reshape(b, hv, n * _CHUNK, dv)[:, :, :t].transpose(1, 2)
    if offsets is not None:
        o = o[inside].unsqueeze(0)
    return o.to(kind), states[:, :, -1]


def _plain_decay_step(q, k, v, g, state, slots):
    kind, group = v.dtype, v.shape[1] // q.shape[1]
    q, k, v = (x.float() for x in (q, k, v))
    q, k = (x.repeat_interleave(group, 1) if group > 1 else x for x in (q, k))
    live = slots >= 0
    at = slots.clamp(min=0).long()
    s = state[at] * g.exp().expand(v.shape[:2])[:, :, None, None] + k[..., None] * v[:, :, None]
    o = (s * q[..., None]).sum(2) * q.shape[-1] ** -0.5
    state[at[live]] = s[live]
    return (o * live[:, None, None]).to(kind)


def _plain_words(seed, site, rows, dim):
    """The generator's words for rows of dim elements, 32 bits each in int64."""
    low = 0xFFFFFFFF
    quads = -(-dim // 4)
    c0 = torch.arange(quads, device=_DEV).expand(rows, quads)
    row = torch.arange(rows, device=_DEV)[:, None].expand(rows, quads)
    c1, c2, c3 = torch.full_like(c0, site), row & low, row >> 32
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57       # modulo 2^64
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, \
            p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], -1).reshape(rows, 4 * quads)[:, :dim]


def _plain_dropout(x, p, seed, site):
    keep = _plain_words(seed, site, *x.shape) >= int(p * 2 ** 32)
    return torch.where(keep, x.float() * (1 / (1 - p)), torch.zeros((), device=_DEV))


def _plain_norm(stream, weight, bias):
    d = stream - stream.mean(-1, keepdim=True)
    return d * torch.rsqrt((d * d).mean(-1, keepdim=True) + _EPS) * weight + bias


def _plain_int4(x, w4, w_scale, bias, group):
    n, k = w4.shape[0], x.shape[-1]
    u = torch.stack([w4 & 15, w4 >> 4], -1).reshape(n, -1)[:, :k].float() - 8
    u = u * w_scale.repeat_interleave(group, 1)[:, :k]
    y = x.float() @ u.t()
    return (y + bias.float() if bias is not None else y).to(x.dtype)


# ------------------------------------------------------------------------------ one pass
def run(s):
    kind, case = s['kind'], s['case']
    if own:
        from brainstate_amd import ops
    if kind == 'decay':
        if own:
            return ops.decay_attention(s['q'], s['k'], s['v'], s['g'], initial_state=s['state'],
                                       seq_offsets=s['offsets'])
        return _plain_decay(s['q'], s['k'], s['v'], s['g'], s['state'], s['offsets'],
                            s['max_len'])
    if kind == 'decay_train':
        args = [s[n].detach().requires_grad_() for n in ('q', 'k', 'v', 'g')]
        with torch.enable_grad():
            if own:
                o = ops.decay_attention(*args, seq_offsets=s['offsets'])[0]
            else:
                o = _plain_decay(*args, None, s['offsets'], s['max_len'])[0]
        return (o.detach(),) + torch.autograd.grad(o, args, s['do'])
    if kind == 'decay_step':
        step = ops.decay_attention_step if own else _plain_decay_step
        o = step(s['q'], s['k'], s['v'], s['g'], s['state'], slots=s['slots'])
        return o, s['state']
    if kind == 'int4':
        linear = ops.int4_linear if own else _plain_int4
        return linear(s['x'], s['w4'], s['w_scale'], bias=s['bias'], group=case['group'])
    if kind == 'norm':
        if own:
            return ops.layer_norm(s['x'], s['weight'], s['bias'], eps=_EPS)
        return _plain_norm(s['x'].float(), s['weight'], s['bias']).to(s['x'].dtype)
    if kind == 'dropout':
        x = s['x'].detach().requires_grad_()
        with torch.enable_grad():
            y = ops.dropout(x, case['p'], s['seed'], site=s['site']) if own else \
                _plain_dropout(x, case['p'], s['seed'], s['site']).to(x.dtype)
        return y.detach(), torch.autograd.grad(y, x, s['dy'])[0]
    args = [s[n].detach().requires_grad_() for n in ('x', 'residual', 'weight', 'bias')]
    with torch.enable_grad():
        if own:
            outs = ops.add_layer_norm(*args, p=case['p'], seed=s['seed'], site=s['site'], eps=_EPS)
        else:
            branch = _plain_dropout(args[0], case['p'], s['seed'], s['site']) if case['p'] else \
                args[0].float()
            stream = args[1].float() + branch
            outs = [t.to(s['x'].dtype) for t in (stream, _plain_norm(stream, *args[2:]))]
    return tuple(t.detach() for t in outs) + torch.autograd.grad(
        outs, args, [s['dstream'], s['dnormed']])


def work(case):
    kind, size = case['kind'], 4 if case['dtype'] == 'f32' else 2
    if kind.startswith('decay'):
        hk, hv, dk, dv, b = (case[n] for n in ('hk', 'hv', 'dk', 'dv', 'batch'))
        n = b * (1 if kind == 'decay_step' else case['tokens'])
        qk, vo = 2 * n * hk * dk * size, 2 * n * hv * dv * size
        gate = 4 * hv * (n if case['each'] else 1)
        cell = n * hv * dk * dv
        if kind == 'decay_step':
            live = b - len(range(0, b, 8)) if b > 8 else b
            return dict(bytes=qk + vo + gate + 8 * live * hv * dk * dv, flops=5 * cell * live // b)
        # the state read and written (2 products of dk x dv a token), and half of the two products
        # within a chunk of 64
        flops = 4 * cell + n * hv * 64 * (dk + dv)
        if kind == 'decay':
            n_seq = case['seqs'] or b
            return dict(bytes=qk + vo + gate + 8 * n_seq * hv * dk * dv, flops=flops)
        # backward: q, k, v, g and the output's gradient in, four gradients out; its products are
        # the state's three and those within a chunk, five
        return dict(bytes=qk + vo + gate + 2 * qk + vo + vo // 2 + 2 * gate, flops=3 * flops)
    if kind == 'int4':
        t, n_in, n_out = case['tokens'], case['n_in'], case['n_out']
        return dict(bytes=t * n_in * size + n_in * n_out // 2 +
                    4 * n_out * -(-n_in // case['group']) + t * n_out * size,
                    flops=2 * t * n_in * n_out)
    n, d = case['rows'] * case['dim'], case['dim']
    if kind == 'norm':
        return dict(bytes=2 * n * size + 8 * d, flops=8 * n)
    if kind == 'dropout':
        return dict(bytes=4 * n * size, flops=4 * n)
    # two operands and two results; the operands, two gradients in, two out (one where nothing is
    # dropped: the operands then have the same gradient)
    return dict(bytes=4 * n * size + 8 * d + n * size * (6 if case['p'] else 5) + 16 * d,
                flops=30 * n)


# ------------------------------------------------------------------------------ in 64 bits
def _exact_decay(q, k, v, g, state, do=None):
    """Token by token in 64 bits, [B, T, H, d] with as many key heads as value heads; with ``do``
    the gradients too, by the recurrence's own transpose."""
    t, scale = q.shape[1], q.shape[-1] ** -0.5
    o = torch.empty_like(v)
    kept = []
    for i in range(t):
        if do is not None:
            kept.append(state)
        state = g[:, i].exp()[..., None, None] * state + k[:, i, :, :, None] * v[:, i, :, None]
        o[:, i] = scale * (state * q[:, i, :, :, None]).sum(2)
    if do is None:
        return o, state
    ds = torch.zeros_like(state)
    dq, dk, dv, dg = (torch.empty_like(x) for x in (q, k, v, g))
    for i in reversed(range(t)):
        ki, vi, doi = k[:, i, :, :, None], v[:, i, :, None], do[:, i, :, None]
        decay = g[:, i].exp()[..., None, None]
        old = decay * kept[i]
        dq[:, i] = scale * ((old + ki * vi) * doi).sum(3)
        ds = ds + scale * q[:, i, :, :, None] * doi
        dk[:, i], dv[:, i] = (ds * vi).sum(3), (ds * ki).sum(2)
        dg[:, i] = (ds * old).sum((2, 3))
        ds = decay * ds
    return o, dq, dk, dv, dg


def _exact_keep(case, s):
    """Which elements dropout keeps, from the generator in numpy's 64-bit unsigned integers."""
    rows, dim, low = case['rows'], case['dim'], np.uint64(0xFFFFFFFF)
    quads, u32 = -(-dim // 4), np.uint64(32)
    x = [np.tile(np.arange(quads, dtype=np.uint64), rows),
         np.full(rows * quads, s['site'], np.uint64),
         np.repeat(np.arange(rows, dtype=np.uint64), quads), np.zeros(rows * quads, np.uint64)]
    key = [s['seed'] % 2 ** 32, s['seed'] // 2 ** 32]
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> u32) ^ x[1] ^ np.uint64(key[0]), b & low,
             (a >> u32) ^ x[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(x, 1).reshape(rows, 4 * quads)[:, :dim]
    return torch.from_numpy(words >= np.uint64(int(case['p'] * 2 ** 32))).to(_DEV)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind.startswith('decay'):
        hk, group = case['hk'], case['hv'] // case['hk']
        x = [s[n].double() for n in ('q', 'k', 'v', 'g')]
        x[:2] = [a.repeat_interleave(group, -2) for a in x[:2]]
        x[3] = x[3].expand(x[2].shape[:-1])
        if kind == 'decay_step':
            x = [a.unsqueeze(1) for a in x]
            state, live = s['state'].double(), s['slots'] >= 0
            at = s['slots'][live].long()
            o = torch.zeros_like(x[2])
            o[live], state[at] = _exact_decay(*(a[live] for a in x), state[at])
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
        if kind == 'decay':
            o, state = _exact_decay(*x, s['state'].double())
            return packed(o), state
        zero = torch.zeros(x[0].shape[0], case['hv'], case['dk'], case['dv'], device=_DEV,
                           dtype=torch.float64)
        if zero.numel() * 8 * x[0].shape[1] > 60e9:
            return None
        r = [packed(a) for a in _exact_decay(*x, zero, side_by_side(s['do'].double()))]
        r[1:3] = [a.reshape(a.shape[:2] + (hk, group, a.shape[3])).sum(3) for a in r[1:3]]
        if not case['each']:
            r[4] = r[4].sum((0, 1))
        return tuple(r)
    if kind == 'int4':
        k, group = case['n_in'], case['group']
        u = torch.empty(case['n_out'], 2 * s['w4'].shape[1], dtype=torch.float64, device=_DEV)
        u[:, ::2], u[:, 1::2] = s['w4'] % 16, s['w4'] // 16
        at = torch.arange(k, device=_DEV) // group
        y = s['x'].double() @ ((u[:, :k] - 8) * s['w_scale'].double()[:, at]).t()
        return y + s['bias'].double() if case['bias'] else y
    x = s['x'].double()
    if kind == 'dropout':
        m = _exact_keep(case, s).double() / (1 - case['p'])
        return x * m, s['dy'].double() * m
    w, b = s['weight'].double(), s['bias'].double()
    m = _exact_keep(case, s).double() / (1 - case['p']) if case.get('p') else torch.ones_like(x)
    stream = s['residual'].double() + x * m if kind == 'norm_train' else x
    mean = stream.mean(1, keepdim=True)
    r = (stream.var(1, unbiased=False, keepdim=True) + _EPS) ** -0.5
    h = (stream - mean) * r
    normed = h * w + b
    if kind == 'norm':
        return normed
    dn = s['dnormed'].double()
    dh = dn * w
    d = s['dstream'].double() + r * (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True))
    return stream, normed, d * m, d, (dn * h).sum(0), dn.sum(0)
