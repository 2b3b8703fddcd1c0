"""Cases of the encoder operators for rotary, windowed and 4-bit layers (rag_enc_qk_norm_rope_dev,
rag_enc_attention_window_dev, rag_enc_linear4_dev): their inputs, one pass through the plain form or through the
framework, the work of a pass and the values in 64 bits."""
import math
import os
import random
import sys

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


_package = None


def _rag():
    global _package
    if _package is None:
        _package = _load()
    return _package


def _load():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'domain-rag-system_amd')
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import rag_hip
    return rag_hip


def listed():
    return [
        # ---- norms of queries and keys + rotation
        # one new token of one query, appended to its kept keys and values: latency
        dict(name='rope_one_token', op='rope', tokens=1, hq=16, hkv=8, d=128, rot=128, inter=False, norm=True, append=4096, type='bf16'),
        # a query batch's tokens (bert-base heads, float32, interleaved pairs over half of the head, no norm)
        dict(name='rope_queries_f32', op='rope', tokens=4001, hq=12, hkv=12, d=64, rot=32, inter=True, norm=False, append=0, type='f32'),
        # packed documents of an indexing batch, grouped heads
        dict(name='rope_documents', op='rope', tokens=16384, hq=32, hkv=8, d=128, rot=128, inter=False, norm=True, append=0, type='bf16'),
        # a large indexing batch, rotation over half of the head
        dict(name='rope_documents_large', op='rope', tokens=65536, hq=16, hkv=8, d=128, rot=64, inter=False, norm=True, append=0, type='f16'),
        # ---- attention with a window and sinks
        # one new token over 2048 kept keys, window 1024: latency
        dict(name='att_one_token', op='att', seqs=1, qlo=1, qhi=1, klo=2048, khi=2048, hq=16, hkv=8, d=128, left=1024, right=0, sinks=4, kept=True, lens=1, type='bf16'),
        # a batch of single tokens over long kept texts, no window: the cache's bytes
        dict(name='att_tokens_long', op='att', seqs=16, qlo=1, qhi=1, klo=4000, khi=32768, hq=32, hkv=8, d=128, left=-1, right=0, sinks=0, kept=True, lens=2, type='f16'),
        # packed passages of up to 512 tokens through a local layer, both directions, first token seen by all
        dict(name='att_passages_local', op='att', seqs=64, qlo=1, qhi=512, klo=0, khi=0, hq=12, hkv=12, d=64, left=64, right=64, sinks=1, kept=False, lens=3, type='bf16'),
        # the same in float32 at the small encoder's heads
        dict(name='att_passages_f32', op='att', seqs=40, qlo=1, qhi=512, klo=0, khi=0, hq=12, hkv=12, d=32, left=128, right=128, sinks=1, kept=False, lens=4, type='f32'),
        # one long document, causal
        dict(name='att_document_long', op='att', seqs=1, qlo=16384, qhi=16384, klo=0, khi=0, hq=16, hkv=8, d=128, left=4096, right=0, sinks=4, kept=False, lens=5, type='bf16'),
        # ---- products with 4-bit weights
        # one token through the small encoder's q|k|v projection, float32 activations: latency
        dict(name='lin_small_f32', op='lin', m=1, n=1152, k=384, group=64, offsets=True, type='f32'),
        # one token through a wide layer
        dict(name='lin_one_token', op='lin', m=1, n=4096, k=4096, group=128, offsets=True, type='bf16'),
        # a query's tokens through a wide layer's expansion, small groups, an odd row count
        dict(name='lin_query', op='lin', m=13, n=16383, k=8192, group=32, offsets=False, type='f16'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(('bf16', 'f16', 'f32'))
    while True:
        op = rng.choice(('rope', 'att', 'lin'))
        if op == 'rope':
            hkv = rng.choice((1, 2, 4, 8, 12))
            d = rng.choice((32, 64, 128))
            c = dict(op='rope', tokens=_log(rng, 1, 65536), hq=hkv * rng.choice((1, 2, 3, 4)), hkv=hkv, d=d, rot=rng.choice((d, d // 2)),
                     inter=rng.random() < 0.5, norm=rng.random() < 0.7, append=0, type=kind)
            if c['tokens'] <= 512 and rng.random() < 0.5:
                c['append'] = 4096
            if c['tokens'] * (c['hq'] + 2 * hkv) * d <= 65536 * 4096:
                return c
        elif op == 'lin':
            group = rng.choice((32, 64, 128))
            c = dict(op='lin', m=_log(rng, 1, 64), n=_log(rng, 64, 16384), k=group * _log(rng, 2, 8192 // group), group=group,
                     offsets=rng.random() < 0.5, type=kind)
            if c['n'] * c['k'] <= 16383 * 8192:
                return c
        else:
            hkv = rng.choice((1, 2, 4, 8))
            c = dict(op='att', hq=hkv * rng.choice((1, 2, 4)), hkv=hkv, d=rng.choice((32, 64, 128)), lens=rng.randrange(1 << 30), type=kind,
                     left=rng.choice((-1, 31, 128, 500, 1024, 4096)), sinks=rng.choice((0, 1, 4, 33)))
            if rng.random() < 0.5:           # tokens over kept keys
                c.update(seqs=_log(rng, 1, 16), qlo=1, qhi=rng.choice((1, 1, 1, 5, 17, 64)), khi=_log(rng, 300, 32768), right=0, kept=True)
                c['klo'] = max(64, c['khi'] // 8)
                cost = c['seqs'] * c['khi'] * max(8 * c['hkv'], c['hq'] * c['qhi'] // 4)
            else:                            # a packed batch
                c.update(seqs=_log(rng, 1, 64), qlo=1, qhi=_log(rng, 16, 8192), klo=0, khi=0, right=rng.choice((0, 0, -1, 64)), kept=False)
                cost = c['seqs'] * c['qhi'] ** 2 * c['hq'] // 128
            if cost <= 16 * 32768 * 64 and c['seqs'] * c['qhi'] * c['hq'] * c['d'] <= 1 << 25:
                return c


# ---- inputs ------------------------------------------------------------------------------------
def _lengths(c):
    """Query and key lengths of a case's sequences, from the case alone."""
    r = random.Random(c['lens'])
    q = [r.randint(c['qlo'], c['qhi']) for _ in range(c['seqs'])]
    k = [max(a, r.randint(c['klo'], c['khi'])) for a in q] if c['kept'] else list(q)
    return q, k


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case['type']]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
    s = dict(case=case)
    if case['op'] == 'rope':
        t, hq, hkv, d, rot = case['tokens'], case['hq'], case['hkv'], case['d'], case['rot']
        s['qkv'] = normal(t, (hq + 2 * hkv) * d).mul_(1.5).to(dt)
        s['inv_freq'] = torch.exp(torch.arange(rot // 2, device=dev, dtype=torch.float64) * (-2 * math.log(10000.0) / rot))
        s['gamma_q'] = (1 + 0.3 * normal(d)).to(dt) if case['norm'] else None
        s['gamma_k'] = (1 + 0.3 * normal(d)).to(dt) if case['norm'] else None
        if case['append']:
            rows = case['append']
            s['k_cache'], s['v_cache'] = normal(rows, hkv, d).to(dt), normal(rows, hkv, d).to(dt)
            s['kv_row'] = torch.randperm(rows, generator=g, device=dev)[:t].contiguous()
            s['pos'] = torch.randint(0, 32768, (t,), generator=g, device=dev, dtype=torch.int32)
        else:
            first = torch.randint(0, 1024, (1,), generator=g, device=dev, dtype=torch.int32)
            s['pos'] = (first + torch.arange(t, device=dev, dtype=torch.int32)).to(torch.int32)
    elif case['op'] == 'att':
        hq, hkv, d = case['hq'], case['hkv'], case['d']
        q_len, k_len = _lengths(case)
        tq = sum(q_len)
        s['cu_q'] = torch.tensor(_starts(q_len), dtype=torch.int32, device=dev)
        s['max_q'], s['max_k'] = max(q_len), max(k_len)
        if case['kept']:
            room = case['khi'] + 16             # every sequence's place among the kept rows
            s['q'] = normal(tq, hq, d).to(dt)
            s['k'] = torch.empty((case['seqs'] * room, hkv, d), dtype=dt, device=dev)
            s['v'] = torch.empty_like(s['k'])
            s['k'].normal_(generator=g)
            s['v'].normal_(generator=g)
            s['k_start'] = torch.arange(case['seqs'], dtype=torch.int64, device=dev) * room
            s['k_len'] = torch.tensor(k_len, dtype=torch.int32, device=dev)
        else:
            qkv = normal(tq, hq + 2 * hkv, d).to(dt)
            s['q'], s['k'], s['v'] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
            s['k_start'], s['k_len'] = None, None
    else:
        m, n, k, group = case['m'], case['n'], case['k'], case['group']
        s['x'] = normal(m, k).to(dt)
        s['codes'] = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)
        step = 0.4 / math.sqrt(k)
        s['scales'] = (step * (0.5 + torch.rand((n, k // group), generator=g, device=dev))).to(dt)
        s['offsets'] = (step * (normal(n, k // group) - 7.5)).to(dt) if case['offsets'] else None
        s['bias'] = normal(n).to(dt)
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(state):
    c = state['case']
    if own:
        rag = _rag()
        if c['op'] == 'rope':
            kw = {}
            if c['append']:
                kw = dict(k_out=state['k_cache'], v_out=state['v_cache'], kv_row=state['kv_row'])
            q, k, v = rag.enc_qk_norm_rope_dev(state['qkv'], state['pos'], state['inv_freq'], c['hq'], c['hkv'], gamma_q=state['gamma_q'],
                                               gamma_k=state['gamma_k'], eps=1e-6, interleaved=c['inter'], **kw)
            return {'q': q, 'k': k, 'v': v} if c['append'] else {'q': q, 'k': k}
        if c['op'] == 'att':
            return rag.enc_attention_window_dev(state['q'], state['k'], state['v'], state['cu_q'], state['max_q'], k_start=state['k_start'],
                                                k_len=state['k_len'], max_k_len=state['max_k'], window_left=c['left'],
                                                window_right=c['right'], n_sinks=c['sinks'])
        return rag.enc_linear4_dev(state['x'], state['codes'], state['scales'], offsets=state['offsets'], bias=state['bias'])
    return {'rope': _plain_rope, 'att': _plain_attention, 'lin': _plain_linear}[c['op']](c, state)


def _plain_rope(c, s):
    t, hq, hkv, d, rot = c['tokens'], c['hq'], c['hkv'], c['d'], c['rot']
    dt = s['qkv'].dtype
    angle = s['pos'].double()[:, None] * s['inv_freq'][None, :]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    x = s['qkv'].float().view(t, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], s['qkv'].view(t, hq + 2 * hkv, d)[:, hq + hkv:]

    def turned(a, gamma):
        if gamma is not None:
            a = a * torch.rsqrt((a * a).mean(dim=-1, keepdim=True) + 1e-6) * gamma.float()
        r = a[..., :rot]
        if c['inter']:
            a0, a1 = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a0 * cos - a1 * sin, a1 * cos + a0 * sin), dim=-1).flatten(-2)
        else:
            a0, a1 = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a0 * cos - a1 * sin, a1 * cos + a0 * sin), dim=-1)
        return torch.cat((r, a[..., rot:]), dim=-1).to(dt)
    q, k = turned(q, s['gamma_q']), turned(k, s['gamma_k'])
    if c['append']:
        s['k_cache'][s['kv_row']] = k
        s['v_cache'][s['kv_row']] = v
        return {'q': q, 'k': s['k_cache'], 'v': s['v_cache']}
    return {'q': q, 'k': k}


def _plain_attention(c, s):
    hq, hkv, d = c['hq'], c['hkv'], c['d']
    n, mq, mk = c['seqs'], s['max_q'], s['max_k']
    dev, dt = s['q'].device, s['q'].dtype
    cu = s['cu_q'].long()
    q_len = cu[1:] - cu[:-1]
    k_len = s['k_len'].long() if s['k_len'] is not None else q_len
    k0 = s['k_start'] if s['k_start'] is not None else cu[:-1]
    jq, jk = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    # padded copies, one row per sequence (a place beyond a sequence's end holds its first row; it is masked)
    iq = cu[:-1, None] + torch.where(jq[None] < q_len[:, None], jq[None], torch.zeros_like(jq[None]))
    ik = k0[:, None] + torch.where(jk[None] < k_len[:, None], jk[None], torch.zeros_like(jk[None]))
    q = s['q'][iq].float().view(n, mq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n * hkv, (hq // hkv) * mq, d)
    k = s['k'][ik].float().permute(0, 2, 3, 1).reshape(n * hkv, d, mk).contiguous()
    v = s['v'][ik].float().permute(0, 2, 1, 3).reshape(n * hkv, mk, d).contiguous()
    p = (k_len - q_len)[:, None, None] + jq[None, :, None]
    key = jk[None, None, :]
    seen = (key < k_len[:, None, None]) & (jq[None, :, None] < q_len[:, None, None])
    if c['right'] >= 0:
        seen &= key - p <= c['right']
    if c['left'] >= 0:
        seen &= (p - key <= c['left']) | (key < c['sinks'])
    score = torch.bmm(q, k).mul_(1 / math.sqrt(d)).view(n, hq, mq, mk)
    score.masked_fill_(~seen[:, None], float('-inf'))
    top = score.amax(dim=-1, keepdim=True)
    score.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = score.sum(dim=-1, keepdim=True)
    out = torch.bmm(score.view(n * hkv, (hq // hkv) * mq, mk), v).view(n, hq, mq, d)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 2, 1, 3)[jq[None] < q_len[:, None]].reshape(-1, hq * d).to(dt)


def _plain_linear(c, s):
    group, k = c['group'], c['k']
    codes = torch.stack((s['codes'] & 15, s['codes'] >> 4), dim=-1).float().view(c['n'], k // group, group)
    scale = s['scales'].float()[:, :, None]
    w = codes * scale + s['offsets'].float()[:, :, None] if s['offsets'] is not None else (codes - 8) * scale
    return (s['x'].float() @ w.view(c['n'], k).t() + s['bias'].float()).to(s['x'].dtype)


# ---- work and exact values ---------------------------------------------------------------------
def _seen_by(j, nq, nk, c):
    """The keys that query j of a sequence sees: the first sinks, then a run [lo, hi)."""
    p = nk - nq + j
    hi = nk if c['right'] < 0 else max(0, min(nk, p + c['right'] + 1))
    lo = 0 if c['left'] < 0 else min(hi, max(0, p - c['left']))
    return min(c['sinks'], lo, hi), lo, hi


def work(case):
    size = 4 if case['type'] == 'f32' else 2
    if case['op'] == 'rope':
        heads = case['hq'] + (2 if case['append'] else 1) * case['hkv']
        elements = case['tokens'] * heads * case['d']
        return {'bytes': 2 * elements * size + 4 * case['tokens'], 'flops': 10 * case['tokens'] * (case['hq'] + case['hkv']) * case['d']}
    if case['op'] == 'att':
        q_len, k_len = _lengths(case)
        pairs = keys = 0
        for nq, nk in zip(q_len, k_len):
            seen = [_seen_by(j, nq, nk, case) for j in range(nq)]
            pairs += sum(a + hi - lo for a, lo, hi in seen)
            first, last = min(lo for _, lo, _ in seen), max(hi for _, _, hi in seen)
            keys += last - first + min(first, case['sinks'])
        return {'bytes': size * case['d'] * (2 * sum(q_len) * case['hq'] + 2 * keys * case['hkv']), 'flops': 4 * pairs * case['hq'] * case['d']}
    m, n, k = case['m'], case['n'], case['k']
    groups = n * (k // case['group']) * (2 if case['offsets'] else 1)
    return {'bytes': n * k // 2 + size * (groups + m * k + m * n + n), 'flops': 2 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'rope':
        t, hq, hkv, d, rot = case['tokens'], case['hq'], case['hkv'], case['d'], case['rot']
        x = s['qkv'].double().view(t, hq + 2 * hkv, d)
        angle = s['pos'].double()[:, None] * s['inv_freq']
        turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]
        done = []
        for part, gamma in ((x[:, :hq], s['gamma_q']), (x[:, hq:hq + hkv], s['gamma_k'])):
            if gamma is not None:
                part = part / torch.sqrt(part.pow(2).sum(dim=-1, keepdim=True) / d + 1e-6) * gamma.double()
            part = part.clone()
            a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case['inter'] else (slice(0, rot // 2), slice(rot // 2, rot))
            z = torch.complex(part[..., a].contiguous(), part[..., b].contiguous()) * turn
            part[..., a], part[..., b] = z.real, z.imag
            done.append(part)
        if not case['append']:
            return {'q': done[0], 'k': done[1]}
        k_all, v_all = s['k_cache'].double(), s['v_cache'].double()
        k_all[s['kv_row']] = done[1]
        v_all[s['kv_row']] = x[:, hq + hkv:]
        return {'q': done[0], 'k': k_all, 'v': v_all}
    if case['op'] == 'att':
        hq, hkv, d = case['hq'], case['hkv'], case['d']
        q_len, k_len = _lengths(case)
        if sum(a * b for a, b in zip(q_len, k_len)) * hq > 16384 * 16384 * 16:
            return None
        at = _starts(q_len)
        out = torch.zeros((at[-1], hq, d), dtype=torch.float64, device=s['q'].device)
        for i, (nq, nk) in enumerate(zip(q_len, k_len)):
            k0 = int(s['k_start'][i]) if case['kept'] else at[i]
            p = torch.arange(nk - nq, nk, device=out.device)[:, None]
            key = torch.arange(nk, device=out.device)[None, :]
            hidden = torch.zeros((nq, nk), dtype=torch.bool, device=out.device)
            if case['right'] >= 0:
                hidden |= key > p + case['right']
            if case['left'] >= 0:
                hidden |= (key < p - case['left']) & (key >= case['sinks'])
            for h in range(hq):
                q = s['q'][at[i]:at[i + 1], h].double()
                k, v = (s[x][k0:k0 + nk, h // (hq // hkv)].double() for x in 'kv')
                score = (q @ k.t() / math.sqrt(d)).masked_fill_(hidden, -math.inf)
                weight = torch.softmax(score, dim=-1)
                out[at[i]:at[i + 1], h] = torch.nan_to_num(weight) @ v
        return out.view(at[-1], hq * d)
    low, high = s['codes'].long() % 16, torch.div(s['codes'].long(), 16, rounding_mode='floor')
    codes = torch.empty((case['n'], case['k']), dtype=torch.float64, device=s['x'].device)
    codes[:, 0::2], codes[:, 1::2] = low.double(), high.double()
    scale = s['scales'].double().repeat_interleave(case['group'], dim=1)
    offset = s['offsets'].double().repeat_interleave(case['group'], dim=1) if case['offsets'] else -8 * scale
    return torch.addmm(s['bias'].double(), s['x'].double(), (codes * scale + offset).t())
