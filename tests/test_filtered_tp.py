"""Sampling filters over a vocabulary in slices: two ranks (gloo, CPU) draw what one process draws from the whole rows, and their
decoders on 4-bit caches shorten the same sequences at the same steps."""
import json
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _check(rank, world, port, out):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from docagents_amd.engine.generator import Generator
    from docagents_amd.models.configs import DecoderConfig
    from docagents_amd.models.llama import LlamaDecoder, TPContext, random_weights, tp_sample
    from docagents_amd.ops import reference as R
    g = torch.Generator().manual_seed(3)
    B, V = 5, 4096
    x = (torch.randn(B, V, generator=g) * 3).bfloat16()
    x[0, 7] = x[0, V - 1] = 30.0
    pos = torch.arange(B, dtype=torch.int32)
    tp = TPContext(rank, world, None)
    part = x[:, rank * V // world:(rank + 1) * V // world].contiguous()
    ok = True
    for f in (dict(top_k=4), dict(top_k=50, top_p=0.9, min_p=0.01), dict(top_p=0.7)):
        a = R.sample_filtered(x, 0.8, 5, ctr=pos, **f)
        b = tp_sample(R, tp, part, 0.8, 5, filters=f, ctr=pos)
        ok &= torch.equal(a[0], b[0]) and torch.allclose(a[1], b[1])
    cfg = DecoderConfig("tiny-4", vocab=512, hidden=256, layers=2, heads=4, kv_heads=2, ffn=128, max_pos=256, rope_theta=1e4)
    w = random_weights(cfg, "cpu", 1, rank, world, full_then_shard=True)
    m = LlamaDecoder(cfg, "cpu", tp=tp, weights=w, kv_bits=4, kv_keep=16, kv_recent=4)
    gen = Generator(m, max_batch=2, max_seq=40, temperature=0.8, check_every=8, top_k=20)
    toks = [r.tokens for r in gen.generate([[3, 5, 7], [2] * 9], 50)]
    all_ = [None] * world
    dist.all_gather_object(all_, (bool(ok), toks))
    if rank == 0:
        with open(out, "w") as f:
            json.dump({"ok": all(o for o, _ in all_), "same": all(t == toks for _, t in all_), "n": [len(t) for t in toks]}, f)
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = tmp_path / "v.json"
    mp.spawn(_check, args=(2, port, str(out)), nprocs=2, join=True)
    v = json.loads(out.read_text())
    assert v["ok"] and v["same"] and v["n"] == [50, 50], v
