"""A Llama / Phi-3 decoder on a 4-bit cache written out in 64 bits: its steps and prompts from the model's weights and from what its
cache holds, with none of the framework's operators. For comparison with the model's own logits.

Tolerance of a comparison. The model rounds to bf16 (half a step: 2^-8) what each of a layer's nine products, norms, rotations and sums
gives, and its last norm and logits: 20 roundings over two layers, which add up to 20 * 2^-8 = 0.078 of the logits' length if they
all point one way."""
import torch

REL = 20 * 2.0 ** -8
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values(codes, scales):
    """[..., D] of codes [..., D / 2] and scales [..., 4]."""
    lut = torch.tensor([*MAGNITUDES, *(-m for m in MAGNITUDES)], dtype=torch.float64)
    codes, scales = codes.cpu().long(), scales.cpu().double()
    x = lut[torch.stack((codes & 15, codes >> 4), -1).flatten(-2)]
    return x * torch.exp2(scales[..., :x.shape[-1] // 32] - 127).repeat_interleave(32, -1)


def loud(m):
    """Weights by which attention decides: random ones give scores near 0, and outputs that the residual drowns."""
    for layer in m.w["layers"]:
        layer["wqkv"].mul_(6)
        layer["wo"].mul_(12)
    return m


def _norm(x, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def _rotated(x, pos, theta):
    """[T, heads, D]: neighbours (2 i, 2 i + 1) by pos theta^(-2 i / D)."""
    D = x.shape[-1]
    a = pos.double()[:, None] * theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    c, s = a.cos()[:, None], a.sin()[:, None]
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack((e * c - o * s, o * c + e * s), -1).flatten(-2)


def forward(m, tokens, pos, attend):
    """Logits [T, vocab]; attend(layer, q [T, H, D], k, v [T, Hkv, D]) -> [T, H, D]. (Gains are folded into the weights.)"""
    c, w = m.cfg, m.w
    D, H, Hkv = c.head_dim, c.heads, c.kv_heads
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    x, pos = d(w["embed"])[tokens.cpu().long()], pos.cpu()
    for li, L in enumerate(w["layers"]):
        y = (_norm(x, c.eps) @ d(L["wqkv"]).t()).view(-1, H + 2 * Hkv, D)
        q, k = _rotated(y[:, :H], pos, c.rope_theta), _rotated(y[:, H:H + Hkv], pos, c.rope_theta)
        x = x + attend(li, q, k, y[:, H + Hkv:]).reshape(len(x), H * D) @ d(L["wo"]).t()
        g = (_norm(x, c.eps) @ d(L["w_gu"]).t()).view(len(x), -1, 2, 16)  # gate and up in rows of 16
        x = x + (torch.nn.functional.silu(g[:, :, 0]) * g[:, :, 1]).flatten(1) @ d(L["w_down"]).t()
    return _norm(x, c.eps) @ d(w["lm_head"]).t()


def _one(q, K, V):
    """q [H, D] over K, V [Hkv, n, D]: outputs [H, D] and each key's probability, summed over the heads of its KV head [Hkv, n]."""
    G = q.shape[0] // K.shape[0]
    p = torch.softmax(torch.einsum("hgd,hnd->hgn", q.view(-1, G, q.shape[1]), K) / q.shape[1] ** 0.5, -1)
    return torch.einsum("hgn,hnd->hgd", p, V).reshape(q.shape), p.sum(1)


def check_step(m, st, rows):
    """One decode step of the model, against the same step written out over the keys that the cache holds after it. The new key's
    codes stand for the written-out key: off by at most a code's half step (1 of the block's units, its largest magnitude is 3.5
    or more of them), plus the model's own roundings."""
    tokens, pos, lens, slot, pre = (t.cpu().clone() for t in (st.tokens, st.pos, st.lens, st.slot, st.pre))
    before = None if m.cache.weight is None else m.cache.weight.cpu().double().clone()
    m.decode_step(st)
    got = st.logits[:rows].cpu().double()
    added = None if before is None else torch.zeros_like(before)
    news = {}

    def attend(li, q, k, v):
        c, out = m.cache.layer(li), torch.zeros_like(q)
        for b in range(rows):
            n, s = int(lens[b]), int(slot[b])
            K, V = (values(x[s, :, :n], y[s, :, :n]) for x, y in ((c.k, c.k_scale), (c.v, c.v_scale)))
            if int(pre[b, 0]):
                P, ps = pre[b].tolist()
                K[:, :P], V[:, :P] = (values(x[ps, :, :P], y[ps, :, :P]) for x, y in ((c.k, c.k_scale), (c.v, c.v_scale)))
            for new, kept in ((k[b], K[:, n - 1]), (v[b], V[:, n - 1])):
                most = new.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
                news[li, b] = bool(((new - kept).abs() <= (1 / 3.5 + REL) * most + REL * new.abs().max()).all())
                assert news[li, b], (li, b)
            out[b], p = _one(q[b], K, V)
            if added is not None:
                added[li, s, :, :n] += p
        return out
    want = forward(m, tokens[:rows], pos[:rows], attend)
    assert len(news) == rows * m.cfg.layers
    err = ((got - want).norm(dim=1) / want.norm(dim=1)).tolist()
    assert max(err) <= REL, err
    if added is not None:
        at = torch.zeros(added.shape, dtype=torch.bool)
        for b in range(rows):
            at[:, slot[b], :, :int(lens[b])] = True
            at[:, slot[b], :, int(lens[b]) - 1] = False  # (written now: what was there is gone)
        diff = (m.cache.weight.cpu().double() - before - added)[at]
        G = m.cfg.heads // m.cfg.kv_heads  # heads whose probabilities a key's weight adds up: REL of 1 each
        assert diff.abs().max() <= REL * G, diff.abs().max()
        assert diff.norm() <= REL * added[at].norm(), (diff.norm(), added[at].norm())
    return want


def prompt_logits(m, prompt, head=None):
    """Logits of a prompt's last token; head (slot, P): behind P keys as that slot holds them."""
    P = 0 if head is None else head[1]

    def attend(li, q, k, v):
        K, V = k.transpose(0, 1), v.transpose(0, 1)
        if P:
            c, s = m.cache.layer(li), head[0]
            K, V = torch.cat((values(c.k[s, :, :P], c.k_scale[s, :, :P]), K), 1), torch.cat((values(c.v[s, :, :P], c.v_scale[s, :, :P]), V), 1)
        return torch.stack([_one(q[t], K[:, :P + t + 1], V[:, :P + t + 1])[0] for t in range(len(prompt))])
    return forward(m, torch.tensor(prompt), P + torch.arange(len(prompt)), attend)[-1]
