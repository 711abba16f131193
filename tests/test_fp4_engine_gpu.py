"""Engines whose layers' matrices are packed into 4 bits (Engine(weights="fp4")), every design: against an engine of the same design
whose bfloat16 matrices hold the values that the packed ones stand for. The two differ by roundings alone, as two orders of sums do: the
bound is the one that bfloat16 engines are held to against the plain implementations."""
import pytest
import torch

from tests.conftest import TINY
from tests.test_bobevik_gpu import MODELS as BOBEVIK, folders as bobevik_folders  # noqa: F401
from tests.test_butolorn_gpu import MODELS as BUTOLORN, folders as butolorn_folders  # noqa: F401
from tests.test_dofipel_gpu import MODELS as DOFIPEL, entry, folders as dofipel_folders, same  # noqa: F401
from tests.test_domorax_gpu import MODELS as DOMORAX, folders as domorax_folders  # noqa: F401
from tests.test_penasun_gpu import MODELS as PENASUN, folders as penasun_folders  # noqa: F401
from tests.test_volonex_gpu import MODELS as VOLONEX, folders as volonex_folders  # noqa: F401

pytestmark = pytest.mark.gpu
DESIGNS = {"bobevik": BOBEVIK, "butolorn": BUTOLORN, "dofipel": DOFIPEL, "domorax": DOMORAX, "penasun": PENASUN, "volonex": VOLONEX}
OPTS = dict(dtype="bfloat16", max_tokens=4096, max_slots=8, max_seq_len=512, beyond_max_positions=True)


def parts_of(model):
    todo = list(model.parts())
    while todo:
        p = todo.pop()
        yield p
        todo += p.children()


def through_four_bits(engine, group):
    """Every matrix that packing would take replaced by the values it would stand for."""
    from hector_engine_amd.kernels import fp4
    from hector_engine_amd.parts.linear import Linear
    from hector_engine_amd.parts.routed import RoutedExperts

    def values(w):
        return fp4.pack(w, group).unpack(w.dtype)
    for p in parts_of(engine.model):
        if isinstance(p, RoutedExperts):
            E, I, S = p.real, p.inter, p.shared_cols
            p.gate_up.weight = values(p.gate_up.weight)
            down = p.down.weight.clone()
            for e in range(E):
                down[:, e * I:(e + 1) * I] = values(down[:, e * I:(e + 1) * I].contiguous())
            if S:
                down[:, E * I:E * I + S] = values(down[:, E * I:E * I + S].contiguous())
            p.down.weight = down
            continue
        for lin in vars(p).values():
            if isinstance(lin, Linear) and lin.packable:
                lin.weight = values(lin.weight)
    return engine


def compare(folder, group, vocab, lengths=(1, 9, 40, 150)):
    import hector_engine_amd as he
    packed = he.Engine(folder, weights="fp4", weight_group=group, **OPTS)
    plain = through_four_bits(he.Engine(folder, **OPTS), group)
    gen = torch.Generator().manual_seed(group)
    for n in lengths:
        ids = torch.randint(0, vocab, (n,), generator=gen).tolist()
        slots = packed.acquire(), plain.acquire()
        want = plain.step([entry(slots[1], ids, range(n))]).clone()
        same(packed.step([entry(slots[0], ids, range(n))]), want.cpu(), "bfloat16")
        packed.release(slots[0])
        plain.release(slots[1])
    # three sequences of different lengths, a prompt joins, one token at a time: eager, captured, replayed
    slots = [(packed.acquire(), plain.acquire()) for _ in range(3)]
    for s, n in zip(slots, (5, 30, 70)):
        ids = torch.randint(0, vocab, (n,), generator=gen).tolist()
        for eng, slot in zip((packed, plain), s):
            eng.step([entry(slot, ids, [n - 1])])
    got, want = [], []
    for _ in range(12):
        ids = torch.randint(0, vocab, (3,), generator=gen).tolist()
        got.append(packed.step([entry(s[0], [t], [0]) for s, t in zip(slots, ids)]).clone())
        want.append(plain.step([entry(s[1], [t], [0]) for s, t in zip(slots, ids)]).clone())
    same(torch.cat(got), torch.cat(want).cpu(), "bfloat16")
    assert packed.stats["graph_replays"] >= 8 and not packed.capture_failures
    return packed


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_the_dense_decoder(model_dirs, name, group):
    from hector_engine_amd.kernels.fp4 import Fp4Weight
    from hector_engine_amd.parts.linear import Linear
    eng = compare(model_dirs[name], group, TINY[name][0]["vocab_size"], (1, 9, 40, 100))
    kinds = [isinstance(lin.weight, Fp4Weight) for p in parts_of(eng.model) for lin in vars(p).values() if isinstance(lin, Linear)]
    assert kinds.count(False) == 1 and kinds.count(True) >= 8      # the head alone is as it was stored


@pytest.mark.parametrize("design", sorted(DESIGNS))
def test_the_other_designs(request, design):
    folders = request.getfixturevalue(f"{design}_folders")
    name = sorted(DESIGNS[design])[0]
    compare(folders[name + "_calm" if name + "_calm" in folders else name], 32, DESIGNS[design][name]["vocab"])


def test_generation_sessions_and_sampling(model_dirs):
    """The paths of a user: generate() step by step and queued give the same ids, a session goes on behind its turns, on packed weights."""
    import hector_engine_amd as he
    eng = he.Engine(model_dirs["D"], weights="fp4", weight_group=32, **OPTS)
    prompts = [[5, 17, 3], [9, 2], list(range(60))]
    a = he.generate(eng, prompts, max_new_tokens=20, stop_ids=())
    b = he.generate(eng, prompts, max_new_tokens=20, stop_ids=(), run_of_steps=1)
    assert [r.tokens for r in a] == [r.tokens for r in b] and all(len(r.tokens) == 20 for r in a)
    session = he.Session(eng, stop_ids=())
    turns = [session.turn([5, 17, 3], 6).tokens, session.turn([8, 8], 6).tokens]
    session.reset()
    assert [session.turn([5, 17, 3], 6).tokens, session.turn([8, 8], 6).tokens] == turns and all(len(t) == 6 for t in turns)


def test_refusals(model_dirs):
    import hector_engine_amd as he
    with pytest.raises(ValueError, match="weights must be"):
        he.Engine(model_dirs["D"], weights="int8", **OPTS)
    with pytest.raises(ValueError, match="go with dtype 'bfloat16'"):
        he.Engine(model_dirs["D"], weights="fp4", **dict(OPTS, dtype="float32"))
    with pytest.raises(ValueError, match="fast kernels"):
        he.Engine(model_dirs["D"], weights="fp4", fast_kernels=False, **OPTS)
    with pytest.raises(ValueError, match="weight_group must be"):
        he.Engine(model_dirs["D"], weights="fp4", weight_group=16, **OPTS)
