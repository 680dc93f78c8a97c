"""``Generator.score`` and ``generate`` check all of a call before it changes a conversation."""
import pytest
import torch

from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import Generator


def _ids(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(0)
    return HybridMoEModel(get_preset("reference_tiny", router_noise_std=0.0, dropout_rate=0.0), compute_dtype=torch.float32).eval()


def _held(gen):
    st = gen.state
    return ([list(st.lengths), list(st.rows), list(st.prefix)], [{n: t.clone() for n, t in c.items()} for c in st.layers.values()],
            st.rows_dev.clone(), st.seen_dev.clone())


CALLS = [("score", dict(sequences=[[1, 2], [3, 512]], prefix=[4, 5]), "token ids of the vocabulary"),
         ("score", dict(sequences=[[1, 2], [3, 4]], prefix=[4, -1]), "token ids of the vocabulary"),
         ("score", dict(sequences=[[1, 2], _ids(21, 1)]), "max_len=20"),
         ("score", dict(sequences=[[1, 2], _ids(21, 1)], prefix=[1]), "max_len=20"),
         ("score", dict(sequences=[[1, 2]], prefix=_ids(21, 1)), "max_len=20"),
         ("score", dict(sequences=[[1, 2], _ids(20, 1)], prefix=_ids(11, 1)), "max_positions=30"),
         ("score", dict(sequences=[[1, 2]], top=65), "top"), ("score", dict(sequences=[[1, 2]], top=-1), "top"),
         ("score", dict(sequences=[[1, 2]], temperature=0.0, prefix=[3]), "temperature"),
         ("generate", dict(prompts=[[1, 2], [3, 512]], max_new_tokens=2, prefix=[4, 5]), "token ids of the vocabulary"),
         ("generate", dict(prompts=[[1, 2], _ids(21, 1)], max_new_tokens=2, prefix=[4, 5]), "max_len=20"),
         ("generate", dict(prompts=[[1, 2], _ids(20, 1)], max_new_tokens=2, prefix=_ids(11, 2)), "max_positions=30"),
         ("generate", dict(prompts=[[1, 2]], max_new_tokens=2, prefix=_ids(31, 2)), "max_"),
         ("prefill", dict(prompts=[[1, 2], [512]], slots=[0, 1]), "token ids of the vocabulary")]


@pytest.mark.parametrize("name,kw,match", CALLS)
def test_refused_calls_leave_every_conversation(model, name, kw, match):
    gen = Generator(model, 4, max_len=20, max_positions=30)
    gen.prefill([_ids(7, 1), _ids(9, 2), _ids(3, 3), _ids(5, 4)], [0, 1, 2, 3])
    kept = _held(gen)
    with pytest.raises(ValueError, match=match):
        getattr(gen, name)(**kw)
    now = _held(gen)
    assert now[0] == kept[0] and torch.equal(now[2], kept[2]) and torch.equal(now[3], kept[3])
    for a, b in zip(now[1], kept[1]):
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_a_shared_slot_is_not_read_into(model):
    gen = Generator(model, 5, max_len=20, max_positions=30)
    gen.prefill([_ids(7, 1)], [0])
    gen.fork(0, [4])
    kept = _held(gen)
    for call in (lambda: gen.score([[1, 2]], prefix=[3]), lambda: gen.generate([[1], [2]], 2, prefix=[3]), lambda: gen.score([[1, 2]])):
        with pytest.raises(ValueError, match="slot 0 is shared"):
            call()
        assert _held(gen)[0] == kept[0]


def test_prompts_as_tensors(model):
    gen = Generator(model, 4, max_len=20, max_positions=30)
    ids = torch.tensor([[1, 2], [3, 4]])
    assert gen.generate(ids, 3, temperature=0.0, prefix=torch.tensor([5, 6]))[0] == gen.generate([[1, 2], [3, 4]], 3, temperature=0.0, prefix=[5, 6])[0]
    assert gen.score(list(ids), prefix=torch.tensor([5])) == gen.score([[1, 2], [3, 4]], prefix=[5])
    assert gen.generate([_ids(40, 1)], 0) == ([[]], [[]])
