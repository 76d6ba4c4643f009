"""The operators of the paged cache, as a list of cases that a timing program can prepare, run and compare.

K and V of every (sequence, kv-head) lie in pages of one chunk each; a table row lists the pages that some later query may still
see.  An entry of a row is (page, position of its first token, last query position that may see it, 0), in the order of positions;
only the last page of a row may be part filled.  A query at position p sees the key at position k of an entry with limit l if k <= p <= l.
With the roles of this package a global or unfinished chunk has no limit, a sliding one c has ``c * P + window + P - 1``, a local one ends with
the next completed global chunk and is open until there is one.

Kinds of cases (``case["kind"]``):

* ``attend``   attention of the last ``n_new`` tokens of every sequence over its pages (their K and V are in them)
* ``roll``     the cache's part of a step: new tokens are written into pages, pages that no later query sees are given back
* ``reorder``  every slot becomes a copy of some slot: replies forked off a prompt, or the survivors of a beam step
* ``step``     all of a step: new tokens into pages, their attention, pages given back

A state can be run again and again: a step appends tokens of sliding chunks only, so that as many pages are taken as are given back.
"""
import math

import numpy as np
import torch

own = False

DEVICE = 'cuda'
GLOBAL, LOCAL, SLIDING = 0, 1, 2
NO_LIMIT, OPEN_LOCAL = 2 ** 31 - 1, 2 ** 31 - 2


def _case(kind, S, Hq, Hkv, D, P, SW, ctx, N, pg, pl, ragged, **more):
    return dict(kind=kind, S=S, Hq=Hq, Hkv=Hkv, D=D, P=P, SW=SW, ctx=ctx, N=N, p_global=pg, p_local=pl, ragged=ragged, **more)


def listed():
    return [
        # one sequence of a small multi-head model, one new token: latency
        dict(_case('attend', 1, 8, 8, 64, 64, 256, 2048, 1, 0.10, 0.30, False), name='attend_token_1'),
        # a decode batch behind prompts of up to 32k tokens, few kept: the bytes of the pages
        dict(_case('attend', 64, 32, 8, 128, 128, 1024, 32768, 1, 0.12, 0.0, True), name='attend_token_64'),
        # up to eight drafted tokens per sequence are checked at once, fine chunks
        dict(_case('attend', 16, 16, 4, 64, 16, 512, 16384, 8, 0.10, 0.15, True), name='attend_draft_16'),
        # a user's short message in a long conversation: few query rows, a long axis of keys
        dict(_case('attend', 2, 32, 8, 128, 32, 1024, 60001, 37, 0.20, 0.10, True), name='attend_message_2'),
        # further turns of several conversations in one padded batch
        dict(_case('attend', 4, 32, 8, 128, 128, 1024, 24576, 1500, 0.10, 0.20, True), name='attend_turn_4'),
        # a segment of a long prompt over the pages of the segments before
        dict(_case('attend', 1, 32, 8, 128, 128, 4096, 131072, 4001, 0.10, 0.08, False), name='attend_segment_131k'),
        # a decode batch's new tokens into pages, expired pages back
        dict(_case('roll', 64, 32, 8, 128, 128, 1024, 8192, 1, 0.05, 0.0, True), name='roll_token_64'),
        # the K and V of a segment of several prompts
        dict(_case('roll', 4, 32, 8, 128, 64, 1024, 16384, 4096, 0.05, 0.0, True), name='roll_segment_4'),
        # eight replies forked off one prompt
        dict(_case('reorder', 8, 32, 8, 128, 128, 1024, 16061, 0, 0.15, 0.0, False, beams=0), name='reorder_replies_8'),
        # a beam step of 16 prompts with four beams each
        dict(_case('reorder', 64, 32, 8, 128, 64, 1024, 12000, 0, 0.10, 0.0, True, beams=4), name='reorder_beams_64'),
        # a whole decode step of a small batch
        dict(_case('step', 16, 32, 8, 128, 64, 1024, 16384, 1, 0.10, 0.0, True), name='step_token_16'),
        # a whole step of a batch that takes prompts in pieces
        dict(_case('step', 8, 16, 8, 64, 32, 512, 8192, 256, 0.10, 0.0, True), name='step_piece_8'),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    rows = case['S'] * case['Hq'] * max(case['N'], 1) if case['kind'] in ('attend', 'step') else 0
    keys = case['ctx'] * (case['p_global'] + case['p_local'] / 4) + 2 * case['SW'] + case['N'] + 4 * case['P']
    return w['flops'] / 1e15 + w['bytes'] / 6e12 + rows * keys / 1e12


def draw(rng):
    largest = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= 0.8 * largest:
            return case


def _draw(rng):
    kind = rng.choice(['attend', 'attend', 'attend', 'attend', 'roll', 'reorder', 'step'])
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([2, 4, 8, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 4, 8])
    P = rng.choice([16, 32, 64, 128, 128])
    SW = P * max(1, _log_uniform(rng, 128, 4096) // P)
    pg, pl = rng.uniform(0.02, 0.20), rng.uniform(0.0, 0.25)
    ragged = rng.random() < 0.7
    if kind == 'attend':
        N = rng.choice([1, 1, _log_uniform(rng, 2, 64), _log_uniform(rng, 64, 4096), _log_uniform(rng, 64, 4096)])
        S = min(64, max(1, _log_uniform(rng, 1, 4096) // N)) if N > 1 else _log_uniform(rng, 1, 96)
        return _case(kind, S, Hq, Hkv, D, P, SW, _log_uniform(rng, 300, 131072 if S <= 4 else 32768), N, pg, pl, ragged)
    if kind == 'roll':
        N = rng.choice([1, _log_uniform(rng, 2, 8192)])
        S = min(64, max(1, _log_uniform(rng, 1, 16384) // N)) if N > 1 else _log_uniform(rng, 1, 96)
        return _case(kind, S, Hkv, Hkv, D, P, SW, _log_uniform(rng, 500, 16384), N, min(pg, 0.1), 0.0, ragged)
    if kind == 'reorder':
        beams = rng.choice([0, 2, 4, 5])
        S = beams * rng.randint(1, 16) if beams else rng.randint(2, 16)
        return _case(kind, S, Hkv, Hkv, D, P, SW, _log_uniform(rng, 500, 16384), 0, pg, 0.0, ragged and beams > 0, beams=beams)
    N = rng.choice([1, 1, _log_uniform(rng, 2, 512)])
    S = min(32, max(1, _log_uniform(rng, 1, 2048) // N)) if N > 1 else _log_uniform(rng, 1, 48)
    return _case(kind, S, Hq, Hkv, D, P, SW, _log_uniform(rng, 500, 16384), N, min(pg, 0.12), 0.0, ragged)


# ---------------------------------------------------------------------------------------------------- preparation
def _lengths(case):
    """Tokens of every sequence in front of its new ones, and how many new ones it has (fixed per case: the same for all seeds)"""
    rng = np.random.default_rng(11)
    S, ctx, N = case['S'], case['ctx'], case['N']
    groups = S // case['beams'] if case.get('beams') else S
    before = rng.integers(max(1, ctx // 3), ctx + 1, groups) if case['ragged'] else np.full(groups, ctx)
    before = np.repeat(before, S // groups)
    new = rng.integers(0 if N > 1 else N, N + 1, S) if case['ragged'] else np.full(S, N)
    if S:
        before[0], new[0] = ctx, N
    if case.get('beams'):
        before[:case['beams']] = ctx
    return before, new


def _limits(roles, total, P, SW):
    """Last query position that may see a chunk, int32 like ``roles``, of sequences of ``total`` [S] tokens"""
    n = roles.shape[-1]
    c = torch.arange(n, device=DEVICE)
    done = ((c + 1) * P <= total[:, None])[:, None]
    closing = torch.where((roles == GLOBAL) & done, c, n)
    after = closing.flip(-1).cummin(-1)[0].flip(-1)                 # the chunk itself or the next completed global one
    limit = torch.where(roles == SLIDING, c * P + SW + P - 1, torch.where(after < n, (after + 1) * P - 1, OPEN_LOCAL))
    return torch.where(done & (roles != GLOBAL), limit, NO_LIMIT).to(torch.int32)


@torch.no_grad()
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    S, Hq, Hkv, D, P, SW, N = (case[k] for k in ('S', 'Hq', 'Hkv', 'D', 'P', 'SW', 'N'))
    kind = case['kind']
    before, new = (torch.from_numpy(x).to(DEVICE) for x in _lengths(case))
    total = before + new if kind == 'attend' else before
    first = before                                                  # pages that no query from here on sees have been given back
    n_chunks = -(-int(total.max()) // P)
    c = torch.arange(n_chunks, device=DEVICE)
    # roles are drawn once per case; the seed decides which (sequence, kv-head) has which
    once = torch.Generator(device=DEVICE).manual_seed(7)
    u = torch.rand(S, Hkv, n_chunks, generator=once, device=DEVICE)
    roles = torch.where(u < case['p_global'], GLOBAL, torch.where(u < case['p_global'] + case['p_local'], LOCAL, SLIDING))
    roles[..., 0] = GLOBAL
    roles = roles[:, torch.randperm(Hkv, generator=g, device=DEVICE)]
    if kind == 'reorder':                                           # replies and beams of a prompt agree in its roles
        b = case['beams'] or S
        roles = roles[::b].repeat_interleave(b, 0)
    limit = _limits(roles, total, P, SW)
    keep = (c * P < total[:, None])[:, None] & (limit >= first[:, None, None])
    n_pages = keep.sum(-1).to(torch.int32)
    per_step = (N + P - 1) // P + 1 if kind in ('roll', 'step') else 0
    if kind in ('roll', 'step'):                                    # room for the steps to come: pages in the window and new ones
        width = int(n_pages.max()) + SW // P + 2 + per_step
    else:
        width = int(n_pages.max()) + 1
    order = torch.argsort((~keep).to(torch.int8), dim=-1, stable=True)[..., :width]
    order = torch.nn.functional.pad(order, (0, width - order.shape[-1]))
    there = torch.arange(width, device=DEVICE) < n_pages[..., None]
    used = int(n_pages.sum())
    spare = S * Hkv * (SW // P + 3 + per_step) if kind in ('roll', 'step') else 2 * S * Hkv
    n_pool = used + spare + 3
    ids = torch.randperm(n_pool, generator=g, device=DEVICE)        # pages of a cache that has been in use for a while
    page = ids[(there.reshape(-1).cumsum(0) - 1).clamp(0).view_as(there)]
    if kind == 'reorder':
        # all slots but the first of a group share the whole pages of the prompt's first half
        b = case['beams'] or S
        shared = there & (order * P < before[:, None, None] // 2)
        page = torch.where(shared, page[::b].repeat_interleave(b, 0), page)
    entries = torch.stack((page, order * P, limit.gather(-1, order), torch.zeros_like(page)), -1) * there[..., None]
    refs = torch.bincount(page[there], minlength=n_pool).to(torch.int32)
    bits = torch.nn.functional.pad((refs == 0).long(), (0, -n_pool % 32)).view(-1, 32)
    bits = (bits << torch.arange(32, device=DEVICE)).sum(-1)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)

    def randn(*shape, sigma=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.bfloat16).mul_(sigma)

    state = dict(case=case, pages_k=randn(n_pool, P, D), pages_v=randn(n_pool, P, D, sigma=0.5), refs=refs, free_bits=bits,
                 entries=entries.to(torch.int32).contiguous(), n_pages=n_pages.contiguous(), length=total.to(torch.int32),
                 n_new=new.to(torch.int32) if case['ragged'] else None)
    if N:
        state['q'] = randn(S, Hq, N, D)
    if kind in ('roll', 'step'):
        state['k'], state['v'] = randn(S, Hkv, N, D), randn(S, Hkv, N, D, sigma=0.5)
        state['roles'] = torch.full((S, Hkv, (N + P - 2) // P + 1), SLIDING, dtype=torch.uint8, device=DEVICE)
    if kind == 'reorder':
        b = case['beams']
        src = torch.zeros(S, device=DEVICE)
        if b:                                                       # survivors of a beam step: some beams twice, some not at all
            group = torch.arange(S, device=DEVICE) // b * b
            src = group + (torch.rand(S, generator=g, device=DEVICE) * b).floor().clamp(max=b - 1)
        state['src'] = src.to(torch.int32)
    return state


# ---------------------------------------------------------------------------------------------------- the plain forms
def _new_tokens(s):
    S, N = s['length'].shape[0], s['case']['N']
    n_new = s['n_new'] if s['n_new'] is not None else torch.full((S,), N, device=s['length'].device)
    return n_new.long()


def _free_bits(refs):
    bits = torch.nn.functional.pad((refs == 0).long(), (0, -refs.numel() % 32)).view(-1, 32)
    bits = (bits << torch.arange(32, device=refs.device)).sum(-1)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)


def _attend(s):
    case = s['case']
    S, Hq, Hkv, D, P, N = (case[k] for k in ('S', 'Hq', 'Hkv', 'D', 'P', 'N'))
    M, dev = s['entries'].shape[2], s['entries'].device
    page, start, limit, _ = s['entries'].long().unbind(-1)
    n_new = _new_tokens(s)
    there = torch.arange(M, device=dev) < s['n_pages'][..., None]
    k = s['pages_k'][page].view(S, Hkv, M * P, D).float()
    v = s['pages_v'][page].view(S, Hkv, M * P, D).float()
    key = (start[..., None] + torch.arange(P, device=dev)).view(S, Hkv, 1, M * P)
    last = torch.where(there, limit, -1).repeat_interleave(P, -1)[:, :, None]
    i = torch.arange(N, device=dev)
    query = torch.where(i < n_new[:, None], s['length'].long()[:, None] - n_new[:, None] + i, -1)[:, None, :, None]
    hidden = ((key > query) | (query > last) | (query < 0))[:, :, None]
    x = torch.matmul(s['q'].float().view(S, Hkv, -1, D), k.transpose(-1, -2)).view(S, Hkv, -1, N, M * P)
    x = x.mul_(D ** -0.5).masked_fill_(hidden, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(S, Hkv, -1, M * P), v).view(S, Hkv, -1, N, D) / total
    return torch.where(total > 0, o, 0).view(S, Hq, N, D).to(s['q'].dtype)


def _append(s):
    case = s['case']
    S, Hkv, P, SW, N = (case[k] for k in ('S', 'Hkv', 'P', 'SW', 'N'))
    dev, entries, M = s['entries'].device, s['entries'], s['entries'].shape[2]
    n_new, old = _new_tokens(s), s['length'].long()
    total = old + n_new
    # the chunks of the call, from the unfinished one on
    i = torch.arange(s['roles'].shape[-1], device=dev)
    c = (old // P)[:, None] + i
    is_there = (c * P < total[:, None])[:, None].expand(-1, Hkv, -1)
    is_new = is_there & (c * P >= old[:, None])[:, None]
    done = ((c + 1) * P <= total[:, None])[:, None]
    closing = torch.where((s['roles'] == GLOBAL) & done, c[:, None], 2 ** 40)
    after = closing.flip(-1).cummin(-1)[0].flip(-1)
    limit = torch.where(s['roles'] == SLIDING, c[:, None] * P + SW + P - 1, torch.where(after < 2 ** 40, (after + 1) * P - 1, OPEN_LOCAL))
    limit = torch.where(done & (s['roles'] != GLOBAL), limit, NO_LIMIT)
    # local chunks of earlier calls end with the first global one
    first = after[..., :1]
    entries[..., 2] = torch.where((entries[..., 2] == OPEN_LOCAL) & (first < 2 ** 40), (first + 1) * P - 1, entries[..., 2].long()).to(torch.int32)
    # pages of the new chunks: the lowest free ones, in the order of slots, heads and chunks
    n_take = is_new.sum()
    free = (s['refs'] == 0).nonzero()[:, 0]
    new = is_new.reshape(-1).nonzero()[:, 0]
    page = torch.zeros(is_new.numel(), dtype=torch.long, device=dev)
    page[new] = free[:n_take]
    s['refs'][free[:n_take]] = 1
    at = s['n_pages'].long()[..., None] + i - (old % P > 0).long()[:, None, None]
    slot, head, chunk = is_there.nonzero().unbind(1)
    at = at[slot, head, chunk]
    page = torch.where(is_new[slot, head, chunk], page.view_as(is_new)[slot, head, chunk], entries[slot, head, at, 0].long())
    row = torch.stack((page, c[slot, chunk] * P, limit[slot, head, chunk], torch.zeros_like(page)), -1)
    entries[slot, head, at] = row.to(torch.int32)
    # the tokens into their pages
    where = torch.zeros(is_there.shape, dtype=torch.long, device=dev)
    where[slot, head, chunk] = page
    t = torch.arange(N, device=dev)
    pos = old[:, None] + t
    seq, tok = (t < n_new[:, None]).nonzero().unbind(1)
    to = where[seq, :, (pos // P - (old // P)[:, None])[seq, tok]]
    at_row = (pos % P)[seq, tok][:, None]
    s['pages_k'][to, at_row] = s['k'][seq, :, tok].to(s['pages_k'].dtype)
    s['pages_v'][to, at_row] = s['v'][seq, :, tok].to(s['pages_v'].dtype)
    s['n_pages'] += is_new.sum(-1).to(torch.int32)
    s['length'] += n_new.to(torch.int32)
    s['free_bits'].copy_(_free_bits(s['refs']))


def _evict(s):
    entries, M = s['entries'], s['entries'].shape[2]
    there = torch.arange(M, device=entries.device) < s['n_pages'][..., None]
    keep = there & (entries[..., 2] >= s['length'][:, None, None])
    gone = entries[..., 0][there & ~keep].long()
    s['refs'].index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    order = torch.argsort((~keep).to(torch.int8), dim=-1, stable=True)
    moved = entries.gather(2, order[..., None].expand(-1, -1, -1, 4))
    n = keep.sum(-1).to(torch.int32)
    entries.copy_(torch.where((torch.arange(M, device=entries.device) < n[..., None])[..., None], moved, entries))
    s['n_pages'].copy_(n)
    s['free_bits'].copy_(_free_bits(s['refs']))


def _reorder(s):
    P, dev = s['case']['P'], s['entries'].device
    S, Hkv, M, _ = s['entries'].shape
    src, slots = s['src'].long(), torch.arange(S, device=dev)
    entries, n_pages, length = s['entries'][src], s['n_pages'][src], s['length'][src]
    part = length % P > 0
    # the unfinished page stays with its own slot, or with the first one that takes it; the others get a copy
    takes = src[None] == slots[:, None]
    keeper = torch.where(src == slots, slots, torch.where(takes, slots, S).amin(1))[src]
    copies = part & (keeper != slots)
    m = torch.arange(M, device=dev)
    there_old, there_new = m < s['n_pages'][..., None], m < n_pages[..., None]
    is_last = there_new & (m == n_pages[..., None] - 1)
    fresh = is_last & copies[:, None, None]
    one = torch.ones((), dtype=torch.int32, device=dev)
    s['refs'].index_add_(0, s['entries'][..., 0][there_old].long(), -one.expand(int(there_old.sum())))
    still = entries[..., 0][there_new & ~fresh].long()
    s['refs'].index_add_(0, still, one.expand(still.numel()))
    old_page = entries[..., 0][fresh].long()
    page = (s['refs'] == 0).nonzero()[:old_page.numel(), 0]
    s['refs'][page] = 1
    row = torch.arange(P, device=dev) < (length % P)[:, None]
    row = row[:, None].expand(-1, Hkv, -1)[fresh.any(-1)]
    for pages in (s['pages_k'], s['pages_v']):
        pages[page] = torch.where(row[..., None], pages[old_page], pages[page])
    entries[..., 0].masked_scatter_(fresh, page.to(torch.int32))
    s['entries'].copy_(torch.where(there_new[..., None], entries, s['entries']))
    s['n_pages'].copy_(n_pages)
    s['length'].copy_(length)
    s['free_bits'].copy_(_free_bits(s['refs']))


# ---------------------------------------------------------------------------------------------------- one pass
@torch.no_grad()
def run(state):
    kind = state['case']['kind']
    if own:
        from neuralattentionsearch_b200 import functional as F
        kv = F.PagedKV(*(state[k] for k in ('pages_k', 'pages_v', 'refs', 'free_bits', 'entries', 'n_pages', 'length')))
        if kind in ('roll', 'step'):
            F.paged_append(kv, state['k'], state['v'], state['roles'], state['case']['SW'], n_new=state['n_new'])
        if kind in ('attend', 'step'):
            o = F.paged_attention(kv, state['q'], n_new=state['n_new'])
        if kind in ('roll', 'step'):
            F.paged_evict(kv)
        if kind == 'reorder':
            F.paged_reorder(kv, state['src'])
    else:
        if kind in ('roll', 'step'):
            _append(state)
        if kind in ('attend', 'step'):
            o = _attend(state)
        if kind in ('roll', 'step'):
            _evict(state)
        if kind == 'reorder':
            _reorder(state)
    if kind == 'attend':
        return o
    tables = [state[k] for k in ('entries', 'n_pages', 'length', 'refs', 'free_bits', 'pages_k', 'pages_v')]
    return [o, *tables] if kind == 'step' else tables


# ---------------------------------------------------------------------------------------------------- 64 bits, work
@torch.no_grad()
def exact(case, seed):
    """Attention of every (sequence, kv-head) by itself, over the keys that a query sees, in 64 bits; in a step the new tokens' K and V
    come straight from the inputs.  Tables and pages are whole numbers and values that are only moved."""
    if case['kind'] not in ('attend', 'step') or work(case)['flops'] > 4e12:
        return None
    s = prepare(case, seed)
    S, Hq, Hkv, D, P, SW, N = (case[k] for k in ('S', 'Hq', 'Hkv', 'D', 'P', 'SW', 'N'))
    G, step = Hq // Hkv, case['kind'] == 'step'
    new, length, n_pages = _new_tokens(s).tolist(), s['length'].tolist(), s['n_pages'].tolist()
    out = torch.zeros(S, Hq, N, D, dtype=torch.float64, device=DEVICE)
    for b in range(S):
        n = new[b]
        old = length[b] if step else length[b] - n
        pos = torch.arange(old, old + n, device=DEVICE)
        for h in range(Hkv if n else 0):
            row = s['entries'][b, h, :n_pages[b][h]].long()
            keys = (row[:, 1:2] + torch.arange(P, device=DEVICE)).flatten()
            ends = row[:, 2].repeat_interleave(P)
            K, V = (s[x][row[:, 0]].reshape(-1, D) for x in ('pages_k', 'pages_v'))
            if step:                                                # new chunks are sliding ones, the unfinished one becomes one
                there = keys < old
                keys, ends = torch.cat((keys[there], pos)), torch.cat((ends[there], pos))
                K, V = torch.cat((K[there], s['k'][b, h, :n])), torch.cat((V[there], s['v'][b, h, :n]))
                chunk = keys // P
                sliding = torch.where((chunk + 1) * P <= old + n, chunk * P + SW + P - 1, NO_LIMIT)
                ends = torch.where(chunk >= old // P, sliding, ends)
            K, V = K.double(), V.double()
            seen = (keys <= pos[:, None]) & (pos[:, None] <= ends)
            for i in range(0, n, 1024):
                q = s['q'][b, h * G:(h + 1) * G, i:i + 1024][:, :n - i].double()
                w = torch.einsum('gnd,kd->gnk', q, K) / math.sqrt(D)
                w = torch.softmax(w.masked_fill(~seen[i:i + 1024], -math.inf), -1).nan_to_num(0.0)
                out[b, h * G:(h + 1) * G, i:i + q.shape[1]] = w @ V
    return [out] + [None] * 7 if step else out


def _expected(case):
    """Per (sequence, kv-head), from a fixed sample of roles: kept tokens in front of the new ones and visible (query, key) pairs"""
    P, SW = case['P'], case['SW']
    before, new = _lengths(case)
    rng = np.random.default_rng(1)
    kept, pairs, picks = 0.0, 0.0, range(0, case['S'], max(1, case['S'] // 8))
    for b in picks:
        n0, n = int(before[b]), int(new[b])
        total, c = n0 + n, np.arange(-(-(n0 + n) // P))
        u = rng.random(len(c))
        role = np.where(u < case['p_global'], GLOBAL, np.where(u < case['p_global'] + case['p_local'], LOCAL, SLIDING))
        role[0] = GLOBAL
        done = (c + 1) * P <= total
        end = np.minimum.accumulate(np.where((role == GLOBAL) & done, c, 2 ** 40)[::-1])[::-1]
        limit = np.where(~done | (role == GLOBAL), NO_LIMIT, np.where(role == SLIDING, c * P + SW + P - 1, np.minimum((end + 1) * P - 1, OPEN_LOCAL)))
        kept += P * float(((c * P < n0) & (limit >= n0)).sum())
        tok = c[:, None] * P + np.arange(P)                          # every key of every chunk: queries in [max(key, n0), min(limit, total - 1)]
        pairs += float(np.clip(np.minimum(limit[:, None], total - 1) - np.maximum(tok, n0) + 1, 0, None)[tok < total].sum())
    return kept / len(picks), pairs / len(picks)


def work(case):
    """Bytes and flops of one pass: 4 * head_dim flops per visible (query, key) pair and query head; q, the kept K and V, the new ones
    and o once; the table rows that a pass has to look at and the pages that it has to copy."""
    kind, S, Hq, Hkv, D, P, N = (case[k] for k in ('kind', 'S', 'Hq', 'Hkv', 'D', 'P', 'N'))
    kept, pairs = _expected(case)
    new = float(_lengths(case)[1].mean()) if N else 0.0
    rows = S * Hkv * 16.0 * (kept / P + 1)
    attend = dict(bytes=S * (2 * Hkv * 2 * D * (kept + new) + 2 * Hq * 2 * D * new) + rows, flops=4.0 * D * S * Hq * pairs)
    roll = 2 * S * Hkv * 2 * 2 * D * new + rows                          # read and written
    if kind == 'attend':
        return attend
    if kind == 'roll':
        return dict(bytes=roll, flops=0)
    if kind == 'reorder':
        tail = float((_lengths(case)[0] % P).mean())
        copies = S - 1 if not case['beams'] else 0.3 * S             # beams that survive twice
        return dict(bytes=2 * rows + copies * Hkv * 2 * 2 * 2 * D * tail, flops=0)
    return dict(bytes=attend['bytes'] + roll, flops=attend['flops'])
