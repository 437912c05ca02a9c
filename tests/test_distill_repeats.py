"""How the distillation finds a token that comes twice among a row's entries, as a model on the CPU:
entries leave their number at two places of a table each, and whichever of those that share a place
holds it in the end, repeated tokens have to be seen."""
import itertools

import pytest


def places(token, low, mixed):
    return token % low, (token * 7 // 3) % mixed


def seen(tokens, holders):
    """The rule of csrc/distill.cu (maybe_twice) for given holders of the places."""
    return any((a != me and (b != me or tokens[a] == t)) or (b != me and tokens[b] == t)
               for me, t in enumerate(tokens) for a, b in [holders(t)])


def by_order(tokens, holders):
    """Held by others in both tables: misses a repeat whose entries hold one place each."""
    return any(holders(t)[0] != me and holders(t)[1] != me for me, t in enumerate(tokens))


def all_outcomes(tokens, low, mixed):
    first, second = {}, {}
    for k, t in enumerate(tokens):
        a, b = places(t, low, mixed)
        first.setdefault(a, []).append(k)
        second.setdefault(b, []).append(k)
    for f in itertools.product(*first.values()):
        for s in itertools.product(*second.values()):
            at, bt = dict(zip(first, f)), dict(zip(second, s))
            yield lambda t: (at[places(t, low, mixed)[0]], bt[places(t, low, mixed)[1]])


@pytest.mark.parametrize("low,mixed", [(2, 3), (3, 3), (5, 4), (1, 1)])
def test_a_repeat_is_seen_whoever_holds_a_place(low, mixed):
    for tokens in itertools.product(range(6), repeat=4):
        repeated = len(set(tokens)) < len(tokens)
        for holders in all_outcomes(tokens, low, mixed):
            assert seen(tokens, holders) or not repeated


def test_the_order_of_stores_cannot_be_relied_on():
    missed = [h for h in all_outcomes((4, 4), 5, 4) if not by_order((4, 4), h)]
    assert missed


def test_a_token_alone_at_its_places_costs_nothing():
    assert not any(seen((0, 1, 2, 3), h) for h in all_outcomes((0, 1, 2, 3), 64, 64))
