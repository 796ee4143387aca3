"""Attention of answers that share prompts at the values, slots and sizes of test_gpu_kv4_edges.py: the same tests with each
lane cut in two, a prompt and an answer's own slots, in caches of their own; and calls at the ends of the caches' sizes."""
import numpy as np
import pytest

import kv4_ref as ref
import test_gpu_kv4_edges as edges
import test_gpu_kv4_shared as shared
from test_gpu_kv4 import Dev, Filled, bf16_randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=70000, seed=None)
    yield e
    e.close()


class Cut:
    """An engine whose attention over a cache takes the slots of each lane from `at` on from a second cache."""

    def __init__(self, eng, at):
        self.eng, self.at, self.made = eng, at, None

    def __getattr__(self, name):
        return getattr(self.eng, name)

    def op_attn_kv4(self, c, layer, lanes, pos, T, q_heads, q, out, *, scale=None, window=0, sinks=0, gate=None):
        import torch
        from qwen35 import KvCache4
        assert not window and not sinks and layer == 0 and min(pos) >= self.at
        if self.made is None or self.made[0] is not c:
            self.close()
            m = c.cap - self.at
            own = KvCache4(self.eng, c.lanes, m, kv_heads=c.kv_heads, head_dim=c.head_dim)
            t = [torch.zeros(c.lanes, c.kv_heads, m, c.head_dim // w, dtype=torch.uint8, device="cuda") for w in (2, 32) * 2]
            torch.cuda.synchronize()
            c.read(0, 0, c.lanes, self.at, m, *[x.data_ptr() for x in t])
            own.write(0, 0, c.lanes, 0, m, *[x.data_ptr() for x in t])
            self.eng.sync()
            self.made = (c, own)
        lanes = np.arange(len(pos)) if lanes is None else np.asarray(lanes)
        self.eng.op_attn_kv4_shared(c, self.made[1], 0, lanes, np.full(len(pos), self.at), lanes, np.asarray(pos) - self.at, T, q_heads,
                                    q, out, scale=scale, gate=gate)

    def close(self):
        if self.made:
            self.made[1].close()
            self.made = None


@pytest.fixture
def cut(engine):
    made = []

    def at(slot):
        made.append(Cut(engine, slot))
        return made[-1]
    yield at
    for c in made:
        c.close()


@pytest.mark.parametrize("hq,kv,d,T,cap,at", [(4, 2, 128, 3, 500, 410), (8, 2, 256, 1, 9000, 8000), (4, 1, 64, 20, 300, 33)])
def test_scores_past_their_spacing(cut, hq, kv, d, T, cap, at):
    edges.test_attention_scores_past_their_spacing(cut(at), hq, kv, d, T, cap)


@pytest.mark.parametrize("hq,kv,d,T,cap,at", [(4, 2, 128, 1, 500, 250), (8, 2, 256, 1, 9000, 1), (8, 2, 256, 1, 9000, 8999), (4, 1, 64, 20, 300, 100)])
def test_largest_values(cut, hq, kv, d, T, cap, at):
    edges.test_attention_largest_values(cut(at), hq, kv, d, T, cap)


@pytest.mark.parametrize("T", [1, 20])
def test_scale_of_zero_and_next_to_it(cut, T):
    edges.test_attention_scale_of_zero_and_next_to_it(cut(170), T)


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (4, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("at,n", [(8997, 6), (4000, 1), (40, 3)])
def test_every_tile(cut, hq, kv, d, at, n):
    """A slot of each of 282 tiles asked for, by one answer or by some that share the prompt, in prompts of nearly all slots,
    of half of them and of few."""
    rng = np.random.default_rng(d + at)
    eng = cut(at)
    P = edges.Pairs(eng, rng, 1, 9001, kv, d, edges.tile_pairs(rng, 282, 9001))
    told = 0
    for i in range(0, 141, hq * n):
        print(f"tiles {hq} {kv} {d} cut at {at}: pairs from {i}", flush=True)
        probe = np.minimum(i + np.arange(hq * n), 140).reshape(n, 1, hq)
        told += P.run(eng, [0] * n, [9000] * n, 1, hq, probe)
    assert told >= 141
    P.f.c.close()


@pytest.mark.parametrize("hq,kv,d,T,lanes,cap,at", [(8, 2, 256, 1, 16, 2000, 1400), (8, 2, 256, 3, 4, 1100, 64), (8, 2, 128, 9, 2, 1500, 1000),
                                                    (6, 1, 64, 12, 1, 5000, 31), (8, 2, 256, 12, 1, 5000, 4000)])
def test_tiles_of_split_rows(cut, hq, kv, d, T, lanes, cap, at):
    edges.test_tiles_of_split_rows(cut(at), hq, kv, d, T, lanes, cap)


def test_rows_past_one_launch(engine):
    """A prompt in pieces: 2,500 rows an answer behind a prompt, more than a launch takes; an answer without one beside it."""
    rng = np.random.default_rng(4)
    T, hq = 2500, 32
    pre, own = Filled(engine, rng, 1, 100, 2, 64), Filled(engine, rng, 4, 2700, 2, 64)
    plane, plen = np.array([0, -1, 0, 0], np.int32), np.array([97, 0, 97, 50], np.int32)
    lanes, pos = np.array([3, 0, 1, 2], np.int32), np.array([200, 0, 13, 32], np.int32)
    got, q, _ = shared.run(engine, pre, own, plane, plen, lanes, pos, T, hq, rng)
    for i in range(4):
        for t in np.r_[0, 1, 2015, 2016, 2017, 2018, T - 1, rng.integers(0, T, 4)]:
            K, V = shared.seen(pre, own, plane[i], plen[i], lanes[i], pos[i] + t + 1)
            r = slice(i * T + t, i * T + t + 1)
            out, pv, big = ref.attention(q[r], K, V, K.shape[1] - 1, 0, 0, 1 / 8)
            want, e = ref.attention_bound(out, pv, big, K.shape[1], 64)
            assert np.all(np.abs(ref.val(got[r]) - want) <= e), (i, t)
    pre.c.close()
    own.c.close()


def test_past_32_bit_offsets(engine):
    """A prompt at the end of a cache of 6.8 GB, answers at the end of another, and rows of q 4 GB apart."""
    import torch
    rng, D, kv, d, cap = np.random.default_rng(16), Dev(), 1024, 64, 32768
    from qwen35 import KvCache4
    big = [KvCache4(engine, 3, cap, kv_heads=kv, head_dim=d) for _ in range(2)]
    K, V = [], []
    for c, m in zip(big, (64, 40)):
        kc, ks, vc, vs = edges.random_rows(rng, 1, kv, m, d)
        t = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
        c.set_len([2], [cap - m])
        torch.cuda.synchronize()
        c.write(0, 2, 1, cap - m, m, *[x.data_ptr() for x in t])
        K.append(ref.values(kc, ks)[0])
        V.append(ref.values(vc, vs)[0])
    qb = bf16_randn(rng, 3, kv, d, scale=0.01)
    ld = 2 ** 31 + 64
    q = torch.zeros(2 * ld + kv * d, dtype=torch.int16, device="cuda")
    for i in range(3):
        q[i * ld:i * ld + kv * d] = D.up(qb[i]).flatten()
    out = torch.zeros(3, kv, d, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    pos = np.array([cap - 40, cap - 9, cap - 1], np.int32)
    engine.op_attn_kv4_shared(big[0], big[1], 0, [2, 2, 2], [cap] * 3, [2] * 3, pos, 1, kv, (q.data_ptr(), ld, d), (out.data_ptr(), kv * d, d))
    engine.sync()
    # the other slots hold zeros: a score of 0, and no V
    g = ref.val(D.bits(out))
    for i in range(3):
        own = pos[i] - (cap - 40) + 1
        k, v = np.concatenate([K[0], K[1][:, :own]], 1), np.concatenate([V[0], V[1][:, :own]], 1)
        s = np.einsum("hd,hnd->hn", ref.val(qb[i]), k) / 8
        w = np.exp(s)
        total = w.sum(1) + cap - 64 + cap - 40
        want = np.einsum("hn,hnd->hd", w, v) / total[:, None]
        mag = np.einsum("hn,hnd->hd", w, np.abs(v)) / total[:, None]
        # weights off by 2^-8, and by 4 * 68 * 2^-24 of a score's size, under 1 here; float32 sums of 65,536; the common weight
        # of the zeros off by 2^-8 in the divisor, and the result's rounding
        assert np.all(np.abs(g[i] - want) <= (2.0 ** -8 + 2.0 ** -15 + 65536 * 2.0 ** -24) * mag + (2.0 ** -8 + 2.0 ** -8) * np.abs(want)), i
    for c in big:
        c.close()
    del q
    torch.cuda.empty_cache()


def test_the_most_lanes(engine):
    """65,535 prompts of a slot each, named from the last on, by two answers each of a cache of as many lanes."""
    import torch
    rng, D, n, d = np.random.default_rng(17), Dev(), 65535, 64
    pre, own = Filled(engine, rng, n, 1, 1, d), Filled(engine, rng, n, 2, 1, d)
    lanes = np.arange(n, dtype=np.int32)
    plane = (n - 1 - lanes // 2).astype(np.int32)
    qb = bf16_randn(rng, n, 1, d)
    q, out = D.up(qb), torch.zeros(n, 1, d, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    engine.op_attn_kv4_shared(pre.c, own.c, 0, plane, np.ones(n), lanes, lanes % 2, 1, 1, (q.data_ptr(), d, d), (out.data_ptr(), d, d))
    engine.sync()
    g = ref.val(D.bits(out))
    for i in np.r_[0, 1, 255, 256, 257, n - 1, rng.integers(0, n, 200)]:
        K, V = shared.seen(pre, own, plane[i], 1, lanes[i], lanes[i] % 2 + 1)
        o, pv, big = ref.attention(ref.val(qb[i:i + 1]), K, V, K.shape[1] - 1, 0, 0, 1 / 8)
        want, e = ref.attention_bound(o, pv, big, K.shape[1], d)
        assert np.all(np.abs(g[i] - want[0]) <= e[0]), i
    pre.c.close()
    own.c.close()
