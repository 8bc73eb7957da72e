"""Plain-PyTorch fp32 reference implementations of every kernel in ``kernels.py``.

Used as the numerics oracle in tests (HIP kernel vs fp32 PyTorch of the same op) and as the
CPU execution path of the models (the container running CPU tests has no GPU). They are NOT a
GPU fallback: on a GPU device the models always call the HIP kernels.
"""
from __future__ import annotations

import math

import numpy as np
import torch
import torch.nn.functional as F

from .cache4 import MAGNITUDES, SCALE_BYTES, Cache4, new_cache4  # noqa: F401

EPI_NONE, EPI_BIAS, EPI_GELU, EPI_SWIGLU, EPI_RESID = 0, 1, 2, 3, 4
EPI_ROPE = 6  # gemm8p only: QKV + RoPE + KV-cache write
EPI_REGLU = 7  # EPI_SWIGLU with relu in place of silu
GATED = (EPI_SWIGLU, EPI_REGLU)


def gemv_fusable(M, N, K, epi=EPI_NONE):
    return M == 1


def gemm(a, w, bias=None, epi=EPI_NONE, resid=None, out=None, rms=None, **_):
    if rms is not None:  # same numerics as rmsnorm() followed by gemm() (bf16 normalised row)
        g = rms[0] if rms[0] is not None else torch.ones(a.shape[1], dtype=a.dtype, device=a.device)
        a = rmsnorm(a, g, rms[1])
    return _epilogue(a.float() @ w.float().t(), w.shape[0], bias, epi, resid, out)


def _epilogue(y, N, bias, epi, resid, out):
    if bias is not None:
        y = y + bias.float()
    if epi == EPI_GELU:
        y = F.gelu(y)
    elif epi in GATED:
        yy = y.view(y.shape[0], N // 32, 2, 16)
        g, u = yy[:, :, 0, :], yy[:, :, 1, :]
        y = ((F.silu(g) if epi == EPI_SWIGLU else F.relu(g)) * u).reshape(y.shape[0], N // 2)
    elif epi == EPI_RESID:
        y = y + resid.float()
    y = y.to(torch.bfloat16)
    if out is not None:
        out.copy_(y)
        return out
    return y


def gemm_f16(a, w, bias=None, epi=EPI_NONE, resid=None, out=None):
    """fp16 oracle of kernels.gemm_f16: fp32 product + epilogue, one fp16 rounding."""
    y = a.float() @ w.float().t()
    if bias is not None:
        y = y + bias.float()
    if epi == EPI_GELU:
        y = F.gelu(y)
    elif epi == EPI_RESID:
        y = y + resid.float()
    y = y.to(torch.float16)
    if out is not None:
        out.copy_(y)
        return out
    return y


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """[F, K] gate + [F, K] up -> [2F, K] rows interleaved in 16-row groups (EPI_SWIGLU layout)."""
    Fd, K = gate.shape
    assert Fd % 16 == 0
    g = gate.view(Fd // 16, 16, K)
    u = up.view(Fd // 16, 16, K)
    return torch.stack([g, u], dim=1).reshape(2 * Fd, K).contiguous()


def rmsnorm(x, w, eps, resid=None, out=None):
    xf = x.float()
    if resid is not None:
        xf = xf + resid.float()
        resid.copy_(xf.to(resid.dtype))
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    y = y.to(x.dtype)
    if out is not None:
        out.copy_(y)
        return out
    return y


def layernorm(x, g, b, eps, resid=None, out=None, fp8_out=False):
    xf = x.float()
    if resid is not None:
        xf = xf + resid.float()
    yf = F.layer_norm(xf, (xf.shape[-1],), g.float(), None if b is None else b.float(), eps)
    y = yf.to(x.dtype)
    if out is not None:
        out.copy_(y)
        y = out
    if fp8_out:
        yq, ys = quant_fp8(yf)
        return y, yq, ys
    return y


def bert_embed_ln(ids, positions, types, word, pos, type_, g, b, eps, out=None, fp8_out=False):
    t = type_[types.long()] if types is not None else type_[0]
    x = word[ids.long()].float() + pos[positions.long()].float() + t.float()
    return layernorm(x.to(word.dtype), g, b, eps, out=out, fp8_out=fp8_out)


def embed(ids, table, out=None):
    y = table[ids.long()]
    if out is not None:
        out.copy_(y)
        return out
    return y


def pool_l2norm(h, cu_seqlens, mode=0, out32=None, out16=None):
    cu = cu_seqlens.tolist()
    rows = []
    for i in range(len(cu) - 1):
        s0, s1 = cu[i], cu[i + 1]
        if mode == 0 or s1 <= s0:
            rows.append(h[s0].float())
        else:
            rows.append(h[s0:s1].float().mean(0))
    v = torch.stack(rows) if rows else torch.zeros((0, h.shape[1]))
    n = v.norm(dim=-1, keepdim=True)
    v = torch.where(n > 0, v / n.clamp_min(1e-30), v)
    if out16 is not None:
        out16.copy_(v.to(out16.dtype))
    if out32 is not None:
        out32.copy_(v)
        return out32
    return v if out16 is None else out16


def rope_table(max_pos: int, D: int, theta: float, device=None) -> torch.Tensor:
    inv = 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    t = torch.arange(max_pos, dtype=torch.float64)
    ang = torch.outer(t, inv)
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous().to(device)


def _rope_rows(x, cs):  # x [T, nh, D], cs [T, D/2, 2]; pairs (2i, 2i+1) rotated by theta_i * pos
    x1, x2 = x[..., 0::2].float(), x[..., 1::2].float()
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).flatten(-2)


def gemm_rope(a, w, pos, cos_sin, H, Hkv, D, slot, k_cache, v_cache, out=None, kv_out=True):
    """QKV projection with RoPE on q / k and the k / v cache write fused (gemm + rope_cache)."""
    qkv = gemm(a, w, out=out)
    return rope_cache(qkv, pos, cos_sin, H, Hkv, D, slot=slot, k_cache=k_cache, v_cache=v_cache)


def rope_cache(qkv, pos, cos_sin, H, Hkv, D, slot=None, k_cache=None, v_cache=None, rotate_q=True):
    T = qkv.shape[0]
    x = qkv.view(T, H + 2 * Hkv, D)
    cs = cos_sin[pos.long()]
    if rotate_q:
        x[:, :H] = _rope_rows(x[:, :H], cs).to(qkv.dtype)
    x[:, H:H + Hkv] = _rope_rows(x[:, H:H + Hkv], cs).to(qkv.dtype)
    if k_cache is not None:
        sl, ps = slot.long(), pos.long()
        k_cache[sl, :, ps] = x[:, H:H + Hkv]
        v_cache[sl, :, ps] = x[:, H + Hkv:]
    return qkv


def flash_kv_cache_ok(D: int, causal: bool) -> bool:
    return causal


def flash_attn_varlen(q, k, v, cu_seqlens, max_seqlen, H, Hkv, D, causal, scale=None, out=None, prefix=None,
                      kv_cache=None):
    """prefix = (k_pre [Hkv, >=P, D], v_pre, P): every sequence's keys are the P shared prefix keys
    followed by its own; query i sits at key position P + i (bottom-right causal).
    kv_cache = (k_cache, v_cache, slot, pos): own keys of the sequence starting at token t read from
    k_cache[slot[t], :, pos[t] + j] (k / v ignored)."""
    if kv_cache is not None:
        kc, vc, ks, kpos = kv_cache
        T = q.shape[0]
        cu = cu_seqlens.tolist()
        k = torch.empty((T, Hkv * D), dtype=q.dtype, device=q.device)
        v = torch.empty((T, Hkv * D), dtype=q.dtype, device=q.device)
        for b in range(len(cu) - 1):
            s0, s1 = cu[b], cu[b + 1]
            if s1 > s0:
                sl, p0 = int(ks[s0]), int(kpos[s0])
                k[s0:s1] = kc[sl, :, p0:p0 + s1 - s0].transpose(0, 1).reshape(s1 - s0, Hkv * D)
                v[s0:s1] = vc[sl, :, p0:p0 + s1 - s0].transpose(0, 1).reshape(s1 - s0, Hkv * D)
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    T = q.shape[0]
    res = torch.empty((T, H * D), dtype=q.dtype, device=q.device)
    cu = cu_seqlens.tolist()
    G = H // Hkv
    P = 0 if prefix is None else int(prefix[2])
    if P:
        kp = prefix[0][:, :P].float().repeat_interleave(G, 0)   # [H, P, D]
        vp = prefix[1][:, :P].float().repeat_interleave(G, 0)
    for b in range(len(cu) - 1):
        s0, s1 = cu[b], cu[b + 1]
        L = s1 - s0
        if L == 0:
            continue
        qq = q[s0:s1, :H * D].float().view(L, H, D).transpose(0, 1)
        kk = k[s0:s1, :Hkv * D].float().view(L, Hkv, D).transpose(0, 1).repeat_interleave(G, 0)
        vv = v[s0:s1, :Hkv * D].float().view(L, Hkv, D).transpose(0, 1).repeat_interleave(G, 0)
        if P:
            kk, vv = torch.cat([kp, kk], 1), torch.cat([vp, vv], 1)
        s = (qq @ kk.transpose(1, 2)) * scale
        if causal:
            m = torch.ones(L, P + L, dtype=torch.bool, device=q.device).triu(P + 1)
            s = s.masked_fill(m, float("-inf"))
        p = s.softmax(-1)
        res[s0:s1] = (p @ vv).transpose(0, 1).reshape(L, H * D).to(q.dtype)
    if out is not None:
        out.copy_(res)
        return out
    return res


def decode_attn(q, k_cache, v_cache, lens, slot, H, Hkv, D, max_len=None, chunk=256, scale=None, out=None, pre=None,
                rope=None):
    """pre: optional int32 [B, 2] = (P, prefix slot): keys [0, P) of row b come from the prefix slot.
    rope = (cos_sin, pos): q is the raw qkv row; RoPE + the new token's cache write happen here
    (rope_cache on a copy of the rows, then attention)."""
    if rope is not None:
        q = rope_cache(q.clone(), rope[1], rope[0], H, Hkv, D, slot=slot, k_cache=k_cache, v_cache=v_cache)
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    B = q.shape[0]
    G = H // Hkv
    res = torch.empty((B, H * D), dtype=q.dtype, device=q.device)
    pre_h = None if pre is None else pre.tolist()
    for b in range(B):
        L, s = int(lens[b]), int(slot[b])
        qq = q[b, :H * D].float().view(H, 1, D)
        kk = k_cache[s, :, :L].float()
        vv = v_cache[s, :, :L].float()
        if pre_h is not None and pre_h[b][0] > 0:
            P, ps = pre_h[b]
            kk = torch.cat([k_cache[ps, :, :P].float(), kk[:, P:]], 1)
            vv = torch.cat([v_cache[ps, :, :P].float(), vv[:, P:]], 1)
        kk, vv = kk.repeat_interleave(G, 0), vv.repeat_interleave(G, 0)
        p = ((qq @ kk.transpose(1, 2)) * scale).softmax(-1)
        res[b] = (p @ vv).reshape(H * D).to(q.dtype)
    if out is not None:
        out.copy_(res)
        return out
    return res


def log_softmax_rows(logits):
    return torch.log_softmax(logits.float(), dim=-1)


_M32 = 0xFFFFFFFF


def _hash_u32(x: np.ndarray) -> np.ndarray:
    """common.h hash_u32 on uint32 arrays (numpy uint32 arithmetic wraps mod 2^32, like the kernel)."""
    x = x ^ (x >> np.uint32(16))
    x = x * np.uint32(0x7feb352d)
    x = x ^ (x >> np.uint32(15))
    x = x * np.uint32(0x846ca68b)
    return x ^ (x >> np.uint32(16))


def gumbel_u01(seed: int, rkey, v) -> np.ndarray:
    """The sampler kernel's counter-based uniform (common.h u01(seed, rkey, v)), bit-exact; rkey and
    v broadcast (uint32-valued integer arrays)."""
    with np.errstate(over="ignore"):
        rk = np.asarray(rkey, dtype=np.uint32)
        vv = np.asarray(v, dtype=np.uint32)
        inner = _hash_u32(vv + np.uint32(0x632be5ab))
        h = _hash_u32(np.uint32(seed & _M32) ^ _hash_u32(rk + np.uint32(0x9e3779b9) * inner))
    return ((h >> np.uint32(8)).astype(np.float64) + 0.5) * (1.0 / 16777216.0)


def _gumbel_scores(x, temperature, seed, rkeys, v0=0):
    """x fp32 [B, V] -> Gumbel-max scores x / T - log(-log u(seed, rkey_b, v0 + v)) (T <= 0: x)."""
    if temperature <= 0:
        return x.double()
    B, V = x.shape
    u = gumbel_u01(seed, rkeys.reshape(B, 1), np.arange(v0, v0 + V, dtype=np.int64).reshape(1, V))
    return x.double().cpu() / temperature - torch.from_numpy(np.log(-np.log(u)))


def _rkeys(B, step, ctr) -> np.ndarray:
    rs = (ctr.cpu().numpy()[:B].astype(np.int64) if ctr is not None else np.full(B, step, dtype=np.int64))
    with np.errstate(over="ignore"):
        return rs.astype(np.uint32) * np.uint32(131071) + np.arange(B, dtype=np.uint32)


def _bookkeep(B, tok, chosen, device, out_tok=None, out_lp=None, conf=None, active=None, pos=None, lens=None,
              hist=None, start=None, eos=()):
    on = active.bool().clone() if active is not None else torch.ones(B, dtype=torch.bool, device=device)
    if out_tok is None:
        out_tok = torch.zeros(B, dtype=torch.int32, device=device)
    out_tok.copy_(torch.where(on, tok, out_tok))
    if out_lp is not None:
        out_lp.copy_(torch.where(on, chosen, out_lp))
    if conf is not None:
        conf[:, 0] += torch.where(on, chosen.exp(), torch.zeros_like(chosen))
        conf[:, 1] += on.float()
    stop = torch.zeros(B, dtype=torch.bool, device=device)
    for e in list(eos)[:4]:
        stop |= tok == e
    if hist is not None:
        gi = (pos - start).long()
        for b in range(B):
            if on[b] and 0 <= gi[b] < hist.shape[1]:
                hist[b, gi[b]] = tok[b]
        stop |= (gi + 1) >= hist.shape[1]
    if pos is not None:
        pos += on.int()
    if lens is not None:
        lens += on.int()
    if active is not None:
        active.copy_(torch.where(on & stop, torch.zeros_like(active), active))
    return out_tok, chosen


def sample(logits, temperature, seed, step=0, out_tok=None, out_lp=None, conf=None, active=None, ctr=None,
           pos=None, lens=None, hist=None, start=None, eos=()):
    """Reference sampler with the kernel's semantics: Gumbel-max at temperature T with the kernel's
    counter-based hash noise (greedy when T <= 0; ties to the lower index), the chosen token's
    log-probability under the untempered distribution, and the device-side bookkeeping."""
    B = logits.shape[0]
    lp = log_softmax_rows(logits)
    sc = _gumbel_scores(logits.float().cpu(), temperature, seed, _rkeys(B, step, ctr))
    tok = sc.argmax(-1).to(logits.device)  # first maximal index = the kernel's lower-index tie rule
    chosen = lp.gather(1, tok.view(-1, 1)).squeeze(1)
    return _bookkeep(B, tok.int(), chosen, logits.device, out_tok, out_lp, conf, active, pos, lens, hist, start, eos)


def sample_filtered(logits, temperature, seed=0, step=0, top_k=0, top_p=1.0, min_p=0.0, u=None, out_tok=None, out_lp=None,
                    conf=None, active=None, ctr=None, pos=None, lens=None, hist=None, start=None, eos=()):
    """See ops.kernels.sample_filtered: row by row, in 64 bits."""
    B, V = logits.shape
    if u is None:
        u = torch.from_numpy(gumbel_u01(seed, _rkeys(B, step, ctr), 0))
    of = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else float(v)  # noqa: E731
    x = logits.double().cpu()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    tok, chosen = torch.zeros(B, dtype=torch.int32), torch.zeros(B)
    for b in range(B):
        z, order = x[b].sort(descending=True, stable=True)
        if z[0] == -math.inf:
            chosen[b] = -math.inf
            continue
        T, k, p, m = of(temperature, b), int(of(top_k, b)), of(top_p, b), of(min_p, b)
        d = torch.where(z == z[0], torch.zeros_like(z), z - z[0])  # (z may be inf)
        n = 1
        if T > 0:
            w = torch.where(d == -math.inf, 0.0, torch.exp(d / T))  # (whatever T, inf among it)
            C = w.cumsum(0)
            n = n_k = k if 0 < k < V else V
            if p < 1:
                n = min(n, int((C < p * C[n_k - 1]).sum()) + 1)
            if m > 0:
                n = min(n, int((w >= m).sum()))
            n = max(n, 1)
        else:
            C = torch.ones(1, dtype=torch.float64)
        at = min(int((C[:n] <= float(u[b]) * C[n - 1]).sum()), n - 1)
        tok[b] = order[at]
        chosen[b] = d[at] - torch.log1p(torch.exp(d[1:]).sum())
    return _bookkeep(B, tok.to(logits.device), chosen.to(logits.device), logits.device, out_tok, out_lp, conf, active, pos, lens,
                     hist, start, eos)


def sample_partial(logits, temperature, seed, v0, step=0, ctr=None, out=None):
    """Vocab-parallel sampling, rank side (see ops.kernels.sample_partial): stats fp32 [B, 8]."""
    B, V = logits.shape
    x = logits.float().cpu()
    sc = _gumbel_scores(x, temperature, seed, _rkeys(B, step, ctr), v0)
    bi = sc.argmax(-1)
    mx = x.max(-1).values
    st = torch.zeros((B, 8), dtype=torch.float32)
    st[:, 0] = sc.gather(1, bi.view(-1, 1)).squeeze(1).float()
    st[:, 1] = (bi + v0).to(torch.int32).view(torch.float32)
    st[:, 2] = mx
    st[:, 3] = torch.exp(x - mx[:, None]).sum(-1)
    st[:, 4] = x.gather(1, bi.view(-1, 1)).squeeze(1)
    st = st.to(logits.device)
    if out is not None:
        out.copy_(st)
        return out
    return st


def sample_finalize(gathered, ranks, out_tok=None, out_lp=None, conf=None, active=None, pos=None, lens=None,
                    hist=None, start=None, eos=()):
    """Vocab-parallel sampling, merge side: gathered [B, ranks * 8] -> sample()'s outputs."""
    B = gathered.shape[0]
    g = gathered.float().cpu().view(B, ranks, 8)
    score, idx = g[..., 0], g[..., 1].contiguous().view(torch.int32).long()
    best = score.max(-1).values
    cand = torch.where(score == best[:, None], idx, torch.full_like(idx, 1 << 40))
    r = cand.argmin(-1)  # max score, ties to the lower global index
    tok = idx.gather(1, r.view(-1, 1)).squeeze(1)
    xb = g[..., 4].gather(1, r.view(-1, 1)).squeeze(1).double()
    gmax = g[..., 2].max(-1).values.double()
    lse = gmax + torch.log((g[..., 3].double() * torch.exp(g[..., 2].double() - gmax[:, None])).sum(-1))
    chosen = (xb - lse).float().to(gathered.device)
    return _bookkeep(B, tok.int().to(gathered.device), chosen, gathered.device, out_tok, out_lp, conf, active, pos,
                     lens, hist, start, eos)


def _found(s, rows, ids):
    return s, rows if ids is None else gather_ids(rows, ids)


def topk_dense(X, Qv, K, thr, slots=None, bitmap=None, ids=None, **_):
    s = Qv.float() @ X.float().t()  # [Q, N]
    valid = s >= thr
    if slots is not None:
        valid &= (slots[:X.shape[0]] >= 0).view(1, -1)
    if bitmap is not None:
        sl = slots[:X.shape[0]].long().clamp_min(0)
        words = bitmap[:, (sl >> 5)]  # [Q, N]
        bits = (words >> (sl & 31).view(1, -1)) & 1
        valid &= bits.bool()
    s = s.masked_fill(~valid, float("-inf"))
    return _found(*_topk_with_ties(s, K), ids)


def _topk_with_ties(s, K):
    Q, N = s.shape
    if N == 0:
        return (torch.full((Q, K), float("-inf")), torch.full((Q, K), -1, dtype=torch.int32))
    # sort desc by score, asc by index
    idx = torch.arange(N, device=s.device).expand(Q, N)
    order = torch.argsort(idx, dim=1, stable=True)
    vals, perm = torch.sort(s, dim=1, descending=True, stable=True)
    ids = torch.gather(idx, 1, perm)
    kk = min(K, N)
    vs, ii = vals[:, :kk], ids[:, :kk].int()
    ii = torch.where(torch.isinf(vs), torch.full_like(ii, -1), ii)
    if kk < K:
        vs = torch.cat([vs, torch.full((Q, K - kk), float("-inf"), device=s.device)], 1)
        ii = torch.cat([ii, torch.full((Q, K - kk), -1, dtype=torch.int32, device=s.device)], 1)
    del order
    return vs, ii


def topk_ranges(X, Qv, ranges, range_off, K, thr, max_rows=None, slots=None, bitmap=None, ids=None, **_):
    Q = Qv.shape[0]
    N = X.shape[0]
    s = Qv.float() @ X.float().t()
    allowed = torch.zeros((Q, N), dtype=torch.bool, device=X.device)
    ro = range_off if isinstance(range_off, list) else range_off.tolist()
    rg = ranges if isinstance(ranges, list) else ranges.reshape(-1).tolist()
    for q in range(Q):
        for r in range(ro[q], ro[q + 1]):
            a, b = rg[2 * r:2 * r + 2]
            allowed[q, a:b] = True
    valid = allowed & (s >= thr)
    if slots is not None:
        valid &= (slots[:N] >= 0).view(1, -1)
    if bitmap is not None:
        sl = slots[:N].long().clamp_min(0)
        bits = (bitmap[:, (sl >> 5)] >> (sl & 31).view(1, -1)) & 1
        valid &= bits.bool()
    s = s.masked_fill(~valid, float("-inf"))
    return _found(*_topk_with_ties(s, K), ids)


def topk_lists(X, Qv, lists, list_off, K, thr, mean_rows=None, max_rows=None, slots=None, bitmap=None, ids=None):
    off = list_off.tolist()
    rg = [[off[x], off[x + 1]] if x >= 0 else [0, 0] for q in lists.tolist() for x in q]
    ro = torch.arange(lists.shape[0] + 1) * lists.shape[1]
    return topk_ranges(X, Qv, torch.tensor(rg).view(-1, 2), ro, K, thr, slots=slots, bitmap=bitmap, ids=ids)


def topk_merge(cand_s, cand_i, K, ids=None):
    P, Q, _ = cand_s.shape
    s = cand_s.permute(1, 0, 2).reshape(Q, -1)
    i = cand_i.permute(1, 0, 2).reshape(Q, -1)
    s = torch.where(i < 0, torch.full_like(s, float("-inf")), s)
    # sort by score desc, id asc
    big = i.clamp_min(0).to(torch.float64)
    key = s.to(torch.float64) * 1e12 - big
    order = torch.argsort(key, dim=1, descending=True, stable=True)
    vs, ii = torch.gather(s, 1, order)[:, :K], torch.gather(i, 1, order)[:, :K]
    ii = torch.where(torch.isinf(vs), torch.full_like(ii, -1), ii)
    return _found(vs, ii, ids)


def gather_ids(rows, ids):
    r = rows.long()
    ok = (r >= 0) & (r < ids.numel())
    return torch.where(ok, torch.nn.functional.pad(ids, (0, 1))[torch.where(ok, r, ids.numel())], torch.full_like(r, -1))


def kmeans_accum(X, assign, sums, counts):
    a = assign.long()
    m = a >= 0
    sums.index_add_(0, a[m], X[m].float())
    counts.index_add_(0, a[m], torch.ones(int(m.sum()), device=X.device))


# ----------------------------------------------------------------------------------- fp8 path
def quant_fp8(x, out=None, scale=None):
    xf = x.float()
    sc = xf.abs().amax(dim=1) / 448.0
    sc = torch.where(sc > 0, sc, torch.ones_like(sc))
    q = (xf / sc[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    if out is not None:
        out.copy_(q)
        q = out
    if scale is not None:
        scale[:sc.numel()].copy_(sc)
        sc = scale
    return q, sc


def gemm_fp8(aq, sa, wq, sw, bias=None, epi=EPI_NONE, resid=None, out=None):
    y = (aq.float() * sa[:aq.shape[0], None].float()) @ (wq.float() * sw[:, None].float()).t()
    return _epilogue(y, wq.shape[0], bias, epi, resid, out)


def quant_weight_fp8(w):
    wf = w.float()
    sw = (wf.abs().amax(dim=1) / 448.0).clamp_min(1e-30)
    return (wf / sw[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).contiguous(), sw.contiguous()


DECODE_DK = True
# above 32 rows the split-K tiles stay faster (bench/midm_chain.py, profiles/r3/dk/): the narrow
# dk tiles re-read the activation block once per 16-64 weight rows
DK_MAX_M = 64
DK_SPLITK_ABOVE = 32


def dk_fusable(M, N, K, epi=EPI_NONE):
    return (DECODE_DK and 2 <= M <= DK_MAX_M and K % 256 == 0 and N % 16 == 0
            and epi in (EPI_NONE, EPI_BIAS, EPI_RESID, *GATED) and (epi not in GATED or N % 32 == 0))


def dk_rope_fits(M, N, K, lda):
    return dk_fusable(M, N, K)


def gemm_dk_rope(a, w, pos, cos_sin, H, Hkv, D, slot, k_cache, v_cache, norm_in=None, out=None, kv_out=True):
    """The QKV projection of gemm_dk.hip: rotation of q / k and the cache write behind the (deferred-norm) product."""
    qkv = gemm_dk(a, w, norm_in=norm_in, out=out)
    return rope_cache(qkv, pos, cos_sin, H, Hkv, D, slot=slot, k_cache=k_cache, v_cache=v_cache)


def dk_parts(N, M=0):
    """gemm_dk.hip dk_fn for EPI_RESID: row-norm partial sums written per output tile; 33..64 rows
    (the split-K route): one per 512 columns (written by the reduce launch)."""
    if DK_SPLITK_ABOVE < M <= 64 and N % 512 == 0:
        return N // 512
    bn = 16 if N <= 4096 else 32 if N <= 8192 else 64
    return (N + bn - 1) // bn


def gemm_dk(a, w, epi=EPI_NONE, bias=None, resid=None, out=None, norm_in=None, ssq_out=None):
    """gemm_dk.hip: optional deferred row RMSNorm of ``a`` from partial sums of squares, then the
    product + epilogue; EPI_RESID may also emit the new rows' per-part sums of squares."""
    M, K = a.shape
    N = w.shape[0]
    x = a.float()
    if norm_in is not None:
        ssq, parts, eps = norm_in
        inv = torch.rsqrt(ssq.view(-1, 64)[:parts, :M].sum(0) / K + eps)
        x = (x * inv[:, None]).to(torch.bfloat16).float()
    y = _epilogue(x @ w.float().t(), N, bias, epi, resid, out)
    if ssq_out is not None:
        parts = dk_parts(N, M)
        bn = -(-N // parts)
        y2 = y.float().pow(2)
        sq = torch.stack([y2[:, i * bn:(i + 1) * bn].sum(-1) for i in range(parts)])  # [parts, M]
        ssq_out.view(-1, 64)[:parts, :M] = sq
    return y


def gemm_resid_norm(a, w, resid, gamma, eps, out=None, h_out=None, bias=None):
    y = gemm(a, w, bias=bias, epi=EPI_RESID, resid=resid)
    (resid if out is None else out).copy_(y)
    h = rmsnorm(y, gamma, eps)
    if h_out is not None:
        h_out.copy_(h)
        return h_out
    return h


# fp16 forms of the encoder ops (kernels.*_f16): these references keep the input dtype
layernorm_f16 = layernorm
bert_embed_ln_f16 = bert_embed_ln
pool_l2norm_f16 = pool_l2norm


def flash_attn_f16(q, k, v, cu_seqlens, max_seqlen, H, Hkv, D, causal=False, scale=None, out=None):
    y = flash_attn_varlen(q.float(), k.float(), v.float(), cu_seqlens, max_seqlen, H, Hkv, D, causal, scale=scale)
    y = y.to(torch.float16)
    if out is not None:
        out.copy_(y)
        return out
    return y


# the batch-of-portions ops (recurrent mixers, paged attention, 32-bit residual stream)
def gemm_ln_fit(M: int, hidden: int, ffn: int) -> bool:
    return False


def encoder_layers_fit(rows: int) -> bool:
    return False


from .seq_reference import (causal_conv, delta_rule, delta_step, delta_step_fits, gated_scan, gemm_any,  # noqa: E402,F401
                            gemm_heads, gemm_partials, latent_attn, latent_flash_fits, latent_prep, partials_fit, rglru_gates, selective_scan,
                            sigmoid_attn, stream_add, stream_final, stream_step)


# ----------------------------------------------------------------------- 4-bit key / value cache
def _encode4(x):
    """[..., D] -> (codes [..., D / 2], scales [..., 4]); csrc/cache4.hip has the format."""
    D = x.shape[-1]
    b = x.float().unflatten(-1, (D // 32, 32))
    bits = b.abs().amax(-1).view(torch.int32)
    e = (((bits + 0x200000) >> 23) - 2).clamp(min=1)
    bad = (bits >> 23) >= 255
    y = (b.double() * torch.exp2(127.0 - e.double()).unsqueeze(-1)).abs()
    # the nearest magnitude, ties to the even code
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    up, down = torch.bucketize(y, mid, right=True), torch.bucketize(y, mid)
    code = torch.where(up % 2 == 0, up, down) | (torch.signbit(b).long() << 3)
    code = code.masked_fill(bad.unsqueeze(-1), 0).flatten(-2).to(torch.uint8)
    scales = torch.zeros((*x.shape[:-1], SCALE_BYTES), dtype=torch.uint8, device=x.device)
    scales[..., :D // 32] = e.masked_fill(bad, 255).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _decode4(codes, scales, dtype=torch.float32):
    D = 2 * codes.shape[-1]
    lut = torch.tensor([*MAGNITUDES, *(-v for v in MAGNITUDES)], dtype=dtype, device=codes.device)
    s = scales[..., :D // 32]
    f = torch.exp2(s.to(dtype) - 127).masked_fill(s == 255, float("nan"))
    x = lut[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    return (x.unflatten(-1, (D // 32, 32)) * f.unsqueeze(-1)).flatten(-2)


def cache4_write(k, v, c, slot, at, weight=None):
    D, T = 2 * c.k.shape[-1], k.shape[0]
    slots, Hkv, max_seq = c.k.shape[-4:-1]
    s, a = slot[:T].long(), at[:T].long()
    ok = (s >= 0) & (s < slots) & (a >= 0) & (a < max_seq)
    s, a = s[ok], a[ok]
    for x, codes, scales in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        codes[s, :, a], scales[s, :, a] = _encode4(x[ok].reshape(-1, Hkv, D))
    if weight is not None:
        weight[s, :, a] = 0.0


def rope_cache4(qkv, pos, cos_sin, H, Hkv, D, slot, at, c, weight=None):
    T = qkv.shape[0]
    ok = (pos[:T] >= 0) & (pos[:T] < cos_sin.shape[0])
    qkv[ok] = rope_cache(qkv[ok], pos[:T][ok], cos_sin, H, Hkv, D)
    cache4_write(qkv[ok][:, H * D:(H + Hkv) * D], qkv[ok][:, (H + Hkv) * D:], c, slot[:T][ok], at[:T][ok], weight)
    return qkv


def cache4_read(c, slot: int, n: int):
    return tuple(_decode4(codes[slot, :, :n], scales[slot, :, :n]).bfloat16() for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)))


def decode_attn4(q, c, lens, slot, H, Hkv, D, max_len=None, scale=None, out=None, pre=None, weight=None, dtype=torch.float32):
    B, G = q.shape[0], H // Hkv
    scale = scale if scale is not None else D ** -0.5
    res = torch.zeros((B, H * D), dtype=q.dtype if dtype == torch.float32 else dtype, device=q.device)
    for b in range(B):
        L, s = int(lens[b]), int(slot[b])
        if L <= 0 or not 0 <= s < c.k.shape[0]:
            continue
        kv = []
        for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
            x = _decode4(codes[s, :, :L], scales[s, :, :L], dtype)
            if pre is not None and int(pre[b, 0]) > 0:
                P, ps = int(pre[b, 0]), int(pre[b, 1])
                x[:, :P] = _decode4(codes[ps, :, :P], scales[ps, :, :P], dtype)
            kv.append(x)
        p = (q[b, :H * D].to(dtype).view(Hkv, G, D) @ kv[0].transpose(1, 2) * scale).softmax(-1)
        res[b] = (p @ kv[1]).reshape(H * D).to(res.dtype)
        if weight is not None:
            weight[s, :, :L] += p.sum(1).to(weight.dtype)
    if out is not None:
        out.copy_(res)
        return out
    return res


def cache4_evict(c, weight, lens, slot, keep: int, recent: int, to=None, out=None, above=None):
    layered = c.k.dim() == 5
    out = torch.empty_like(lens) if out is None else out
    to = slot if to is None else to
    for b in range(lens.numel()):
        n, s, d = int(lens[b]), int(slot[b]), int(to[b])
        n_kept = min(n, keep) if n > (keep if above is None else above) else n
        out[b] = n_kept
        for layer in range(c.k.shape[0] if layered else 1):
            w = (weight[layer] if layered else weight)
            one = c.layer(layer) if layered else c
            for h in range(c.k.shape[-3]):
                pick = torch.arange(n, device=w.device)
                if n > n_kept:
                    m = n - recent
                    x = w[s, h, :m]
                    x = torch.where(x.isnan(), torch.full_like(x, float("-inf")), x)
                    # NaN least: behind the others of weight -inf
                    order = torch.argsort(x, descending=True, stable=True)
                    order = torch.cat((order[~w[s, h, :m][order].isnan()], order[w[s, h, :m][order].isnan()]))
                    pick = torch.cat((order[:keep - recent].sort()[0], pick[m:]))
                for t in (*one, w):
                    t[d, h, :len(pick)] = t[s, h, pick].clone()
    return out
