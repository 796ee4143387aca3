"""The operators of answers that share a prompt in a run as they are used: a prompt of text and picture patches appended at
positions on three axes, answers appended behind it a token a round, their attention over prompt and own slots, logits, and the log
probabilities of the tokens that go on. Each stage against float64 on the bits that it read (test_gpu_kv4_axes.py,
test_gpu_kv4_shared.py and test_gpu_logprobs.py say with which tolerances); the rounds enqueue the engine's calls without
waits between them."""
import numpy as np
import pytest

import kv4_ref as ref
import test_gpu_kv4_shared as shared
import test_gpu_logprobs as lp
from test_gpu_kv4 import Dev, bf16_randn, read_cache
from test_gpu_kv4_axes import close, turned

pytestmark = pytest.mark.gpu

HQ, KV, D, ROT, THETA, EPS, VOCAB, TOP = 8, 2, 256, 64, 1e7, 1e-6, 5003, 6
PROMPTS, EACH, ROUNDS = [150, 33], 5, 4


class Bed:
    """A layer's weights and caches, and the run of PROMPTS' answers."""

    def __init__(self, eng, rng):
        import torch
        from qwen35 import KvCache4, pair_axes
        self.eng, self.torch, self.axis = eng, torch, pair_axes([11, 11, 10], True)
        self.pre = KvCache4(eng, len(PROMPTS), 200, kv_heads=KV, head_dim=D)
        self.own = KvCache4(eng, len(PROMPTS) * EACH, 40, kv_heads=KV, head_dim=D)
        self.width = (2 * HQ + 2 * KV) * D
        self.qn, self.kn = bf16_randn(rng, D, scale=0.1), bf16_randn(rng, D, scale=0.1)
        up = Dev().up
        self.qn_d, self.kn_d = up(self.qn), up(self.kn)
        self.table = up(bf16_randn(rng, VOCAB, self.width)).view(torch.bfloat16)       # a token's projections
        self.head = up(bf16_randn(rng, VOCAB, HQ * D, scale=0.05)).view(torch.bfloat16)
        self.prompts = [torch.from_numpy(rng.integers(0, VOCAB, n)).cuda() for n in PROMPTS]
        # a picture of 4 x 6 patches behind 20 tokens: one place in time, rows and columns of their own
        self.places = []
        for n in PROMPTS:
            t = np.arange(n)
            at = np.stack([t, t, t], 1)
            patch = (t >= 20) & (t < 44)
            at[patch] = 20 + np.stack([0 * t, (t - 20) // 6, (t - 20) % 6], 1)[patch]
            at[t >= 44] -= 24 - 6
            self.places.append(at.astype(np.int32))

    def views(self, x):
        p, w = x.data_ptr(), self.width
        return {"q": (p, w, 2 * D), "k": (p + 4 * HQ * D, w, D), "v": (p + 2 * (2 * HQ + KV) * D, w, D)}

    def append(self, cache, lanes, slots, T, x, at, q_out):
        self.eng.op_kv4_append_axes(cache, 0, lanes, slots, T, HQ, (at.data_ptr(), 3, 1), self.axis, rot_dim=ROT, theta=THETA,
                                    eps=EPS, q_norm=self.qn_d.data_ptr(), k_norm=self.kn_d.data_ptr(),
                                    q_out=(q_out.data_ptr(), HQ * D, D), **self.views(x))

    def run(self):
        t = self.torch
        n = len(PROMPTS) * EACH
        zero = np.zeros(n, np.int32)
        for c, m in ((self.pre, len(PROMPTS)), (self.own, n)):
            c.set_len(None, np.zeros(m, np.int32))
        at = [t.from_numpy(a).cuda() for a in self.places]
        x = [self.table[p] for p in self.prompts]
        q = [t.zeros(len(p), HQ, D, dtype=t.int16, device="cuda") for p in self.prompts]
        t.cuda.synchronize()
        for i, m in enumerate(PROMPTS):
            self.append(self.pre, np.array([i], np.int32), np.zeros(1, np.int32), m, x[i], at[i], q[i])
        plane = np.repeat(np.arange(len(PROMPTS)), EACH).astype(np.int32)
        plen = np.array(PROMPTS, np.int32)[plane]
        nxt = np.array([a[-1].max() + 1 for a in self.places])[plane]
        lanes = np.arange(n, dtype=np.int32)[::-1].copy()
        tok = t.arange(n, device="cuda") * 17 + 3
        log = []
        for r in range(ROUNDS):
            x = self.table[tok].contiguous()
            a = t.from_numpy(np.repeat(nxt + r, 3).reshape(n, 3).astype(np.int32)).cuda()
            qo, out = (t.zeros(n, HQ, D, dtype=t.int16, device="cuda") for _ in range(2))
            t.cuda.synchronize()
            self.append(self.own, lanes, zero + r, 1, x, a, qo)
            self.eng.op_attn_kv4_shared(self.pre, self.own, 0, plane, plen, lanes, zero + r, 1, HQ, (qo.data_ptr(), HQ * D, D),
                                        (out.data_ptr(), HQ * D, D), gate=(x.data_ptr() + 2 * D, self.width, 2 * D))
            self.eng.sync()
            logits = out.view(t.bfloat16).view(n, HQ * D).float() @ self.head.float().t()
            tok = logits.topk(3, 1).indices[t.arange(n, device="cuda"), t.arange(n, device="cuda") % 3]
            tg = tok.int()
            got = {k: t.zeros(n, *s, dtype=d, device="cuda") for k, s, d in
                   [("logprobs", (), t.float32), ("ranks", (), t.int32), ("entropy", (), t.float32), ("top_ids", (TOP,), t.int32),
                    ("top_logprobs", (TOP,), t.float32)]}
            t.cuda.synchronize()
            self.eng.op_token_logprobs(n, VOCAB, logits.data_ptr(), targets=tg.data_ptr(), top=TOP,
                                       **{k: v.data_ptr() for k, v in got.items()})
            self.eng.sync()
            log.append(dict(x=x, at=a.cpu().numpy(), q=Dev().bits(qo), out=Dev().bits(out), logits=logits.cpu().numpy(),
                            tok=tg.cpu().numpy(), **{k: v.cpu().numpy() for k, v in got.items()}))
        return plane, plen, lanes, log


class Held:
    """What a cache's lanes hold, as float64 values."""

    def __init__(self, eng, c, lanes, m):
        self.c = c
        kc, ks, vc, vs = read_cache(eng, c, 0, 0, lanes, 0, m)
        self.K, self.V = ref.values(kc, ks), ref.values(vc, vs)


def test_run():
    from qwen35 import Engine
    eng = Engine(max_rows=16, max_ctx=256, seed=None)
    try:
        b = Bed(eng, np.random.default_rng(3))
        plane, plen, lanes, log = b.run()
        again = b.run()[3]
        pre, own = Held(eng, b.pre, len(PROMPTS), min(PROMPTS)), Held(eng, b.own, lanes.size, ROUNDS)
        long = Held(eng, b.pre, 1, PROMPTS[0])
        pre.K, pre.V = [long.K[0], pre.K[1]], [long.V[0], pre.V[1]]
        n = lanes.size
        for r, s in enumerate(log):
            print(f"round {r}", flush=True)
            for k, v in s.items():
                assert k == "x" or np.array_equal(v, again[r][k]), k
            x = ref.val(s["x"].view(b.torch.int16).cpu().numpy().view(np.uint16))
            qg = x[:, :2 * HQ * D].reshape(n, HQ, 2 * D)
            close(s["q"], *turned(qg[..., :D], b.qn, s["at"], b.axis, ROT, THETA, EPS))
            shared.check(pre, own, plane, plen, lanes, np.full(n, r), 1, s["out"], ref.val(s["q"]), qg[..., D:])
            lp.check(s, s["logits"], s["tok"], TOP)
            assert np.array_equal(s["ranks"], np.arange(n) % 3)
    finally:
        eng.close()
