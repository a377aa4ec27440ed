"""A cache in 8 bits under the traffic of an engine: prompts with shared prefixes, decode steps from graphs of padded batches,
sequences that end or are put off while others take over their blocks, rows and scales and all."""
import pytest
import torch

from fp8_cases import assert_within, prefill_reference, to_codes
from nano_vllm_b200 import _lib, attention as A, context as C
from oracle import fp8_cache_ref as F8

pytestmark = pytest.mark.gpu


class Server:
    WIDTH = 4

    def __init__(self, cuda, seed, blocks, hq, hkv, d):
        self.cuda, self.hq, self.hkv, self.d, self.scale = cuda, hq, hkv, d, d ** -0.5
        self.gen = torch.Generator().manual_seed(seed)
        self.layer = A.Attention(hq, d, self.scale, hkv)
        self.ref = [torch.randint(0, 256, (blocks, 256, hkv, d), generator=self.gen, dtype=torch.uint8) for _ in range(2)]
        self.ref += [torch.exp2(torch.randint(-9, 9, (blocks, hkv, 16), generator=self.gen).float()) for _ in range(2)]  # of earlier owners
        self.layer.k_cache, self.layer.v_cache = (t.to(cuda).view(torch.float8_e4m3fn) for t in self.ref[:2])
        self.layer.k_scale, self.layer.v_scale = (t.to(cuda) for t in self.ref[2:])
        self.free, self.users = list(range(blocks)), [0] * blocks
        self.tables, self.lens = {}, {}  # of the sequences that run
        i32 = dict(dtype=torch.int32, device=cuda)
        self.graphs = {}
        for size in (2, 4, 8):
            s = dict(qkv=torch.zeros(size, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=cuda), slots=torch.full((size,), -1, **i32),
                     lens=torch.zeros(size, **i32), tables=torch.zeros(size, self.WIDTH, **i32), graph=torch.cuda.CUDAGraph())
            C.set_context(False, slot_mapping=s["slots"], context_lens=s["lens"], block_tables=s["tables"])
            with torch.cuda.graph(s["graph"]):
                s["out"] = self.layer(*self.split(s["qkv"]))
            self.graphs[size] = s
        C.reset_context()

    def split(self, qkv):
        return qkv.split([self.hq * self.d, self.hkv * self.d, self.hkv * self.d], dim=-1)

    def rows(self, n):
        """A step's activations: tokens differ in size by far more than a scale's binade."""
        qkv = torch.randn(n, (self.hq + 2 * self.hkv) * self.d, generator=self.gen)
        qkv[:, self.hq * self.d:] *= torch.exp(1.5 * torch.randn(n, 1, generator=self.gen))
        q, k, v = self.split(qkv.bfloat16())
        return qkv.bfloat16(), q.view(n, self.hq, self.d), k.view(n, self.hkv, self.d), v.view(n, self.hkv, self.d)

    def grow(self, name, length):
        table = self.tables.setdefault(name, [])
        while len(table) * 256 < length:
            table.append(self.free.pop())
            self.users[table[-1]] += 1
        self.lens[name] = length

    def end(self, *names):
        for name in names:
            for b in self.tables.pop(name):
                self.users[b] -= 1
                if self.users[b] == 0:
                    self.free.append(b)  # the next to be taken
            del self.lens[name]

    def slots(self, name, first, last):
        return [self.tables[name][p // 256] * 256 + p % 256 for p in range(first, last)]

    def table_rows(self, names):
        return torch.tensor([self.tables[n] + [-1] * (self.WIDTH - len(self.tables[n])) for n in names], dtype=torch.int32)

    def prompts(self, *wanted):
        """wanted: (name, new tokens, name of a running sequence whose first full blocks it shares or None, how many)."""
        new, cached, slots = [], [], []
        for name, n, parent, shared in wanted:
            self.tables[name] = list(self.tables[parent][:shared]) if parent else []
            for b in self.tables[name]:
                self.users[b] += 1
            start = 256 * len(self.tables[name])
            self.grow(name, start + n)
            new.append(n)
            cached.append(start)
            slots += self.slots(name, start, start + n)
        names = [w[0] for w in wanted]
        cu_q = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        cu_k = torch.tensor([0] + [a + b for a, b in zip(new, cached)]).cumsum(0).to(torch.int32)
        slots, tables = torch.tensor(slots, dtype=torch.int32), self.table_rows(names) if any(cached) else None
        C.set_context(True, cu_q.to(self.cuda), cu_k.to(self.cuda), max(new), int(cu_k.diff().max()), slots.to(self.cuda), None,
                      tables.to(self.cuda) if any(cached) else None)
        qkv, q, k, v = self.rows(sum(new))
        out = self.layer(*self.split(qkv.to(self.cuda))).view(-1, self.hq, self.d)
        C.reset_context()
        F8.store_kvcache_fp8_ref(k, v, *self.ref, slots)
        if any(cached):
            assert_within(out, *prefill_reference(q, self.ref, cu_q, cu_k, tables, self.scale), names)
        else:
            for a, b in zip(cu_q.tolist(), cu_q.tolist()[1:]):
                ref, bound = F8.attend(q[a:b], k[a:b], v[a:b], self.scale, torch.ones(b - a, b - a).tril().bool())
                assert_within(out[a:b], ref, 6 * bound, names)  # P in bf16: 2^-8 A, where the bound has 1.5 * 2^-11 A
        self.same()

    def decode(self, steps):
        for _ in range(steps):
            names = sorted(self.lens)
            for name in names:
                self.grow(name, self.lens[name] + 1)
            n = len(names)
            s = self.graphs[min(k for k in self.graphs if k >= n)]
            size = len(s["slots"])
            slots = torch.tensor([self.slots(b, self.lens[b] - 1, self.lens[b])[0] for b in names] + [-1] * (size - n), dtype=torch.int32)
            ctx = torch.tensor([self.lens[b] for b in names] + [0] * (size - n), dtype=torch.int32)
            tables = torch.zeros(size, self.WIDTH, dtype=torch.int32)
            tables[:n] = self.table_rows(names)
            qkv, q, k, v = self.rows(size)
            for key, t in (("qkv", qkv), ("slots", slots), ("lens", ctx), ("tables", tables)):
                s[key].copy_(t)
            s["graph"].replay()
            F8.store_kvcache_fp8_ref(k, v, *self.ref, slots)
            assert_within(s["out"].view(size, self.hq, self.d), *F8.decode_fp8_ref(q, *self.ref, ctx, tables, self.scale), names)
        self.same()

    def same(self):
        layer = self.layer
        for got, want in zip((to_codes(layer.k_cache), to_codes(layer.v_cache), layer.k_scale.cpu(), layer.v_scale.cpu()), self.ref):
            assert torch.equal(got, want)
        assert _lib.read_status() == 0


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (14, 2, 64)])
def test_traffic(cuda, hq, hkv, d):
    s = Server(cuda, hq, 14, hq, hkv, d)
    s.prompts(("a", 300, None, 0), ("b", 700, None, 0), ("c", 255, None, 0))
    s.decode(5)                                              # a, b, c in a batch of four; c into its second block
    s.prompts(("d", 30, "b", 2), ("e", 1, "b", 1), ("f", 90, None, 0))  # behind shared blocks, and one beside them
    s.decode(20)                                             # six of eight
    s.end("b", "f")                                          # d and e still hold b's first blocks
    s.decode(3)
    s.prompts(("g", 512, None, 0), ("h", 3, "d", 2))         # in b's and f's blocks, dirty as they are
    s.decode(12)
    put_off = s.lens["a"]
    s.end("a", "e")
    s.prompts(("i", 17, None, 0))
    s.decode(2)
    s.end("i")
    s.prompts(("a", put_off, None, 0))                       # all of its tokens anew, elsewhere
    s.decode(18)
    s.end("c", "d", "g")
    s.decode(2)                                              # two left, in the smallest graph
    s.end(*list(s.lens))
    assert sorted(s.free) == list(range(14)) and not any(s.users)
