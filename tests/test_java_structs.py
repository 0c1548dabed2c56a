"""The argument structs of a block of experts as the Java module lays them out (no JDK here compiles it): sizes, offsets and types are those of
the C structs, and a block's type is the caller's to say."""
from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

import pytest

from jax4j_amd import _native as N

JAVA = Path(__file__).resolve().parents[1] / "java/src/main/java/com/nablatensor/jax4j/backend/mi355x"
SIZES = {"LONG": 8, "INT": 4, "FLOAT": 4}
STRUCTS = [("Mi355xBackend", "NORM_INTO", N.NormArgs), ("Mi355xBackend", "ROUTE_INTO", N.RouteArgs), ("Mi355xExperts", "EXPERTS_APPLY", N.ExpertsArgs),
           ("Mi355xExperts", "return s;", N.NormKind), ("Mi355xExperts", "activation.ordinal()", N.ExpertsConfig)]


def written(source, end):
    """{offset: (type, value)} and the bytes allocated, of the struct that is filled last before `end`."""
    text = (JAVA / f"{source}.java").read_text()
    part = text[:text.index(end) + len(end) + 4]
    part = part[part.rindex("a.allocate("):]
    size = int(re.match(r"a\.allocate\((\d+), 8\)", part)[1])
    return size, {int(at): (kind, value) for kind, at, value in re.findall(r"s\.set\(JAVA_(\w+), (\d+), (.+?)\);", part)}


@pytest.mark.parametrize("source,end,struct", STRUCTS)
def test_layout(source, end, struct):
    size, sets = written(source, end)
    assert C.sizeof(struct) <= size < C.sizeof(struct) + 16
    fields = {getattr(struct, name).offset: (name, kind) for name, kind in struct._fields_}
    assert sets
    for at, (kind, value) in sets.items():
        name, ctype = fields[at]
        assert C.sizeof(ctype) == SIZES[kind] and (ctype is C.c_float) == (kind == "FLOAT"), (name, kind, value)


def test_a_block_s_type_is_the_caller_s():
    """What applyBf16 writes is a block that norm can be told of; read as F32 it would be twice as long as it is."""
    _, sets = written("Mi355xBackend", "NORM_INTO")
    assert sets[N.NormArgs.block_type.offset][1] == "blockBf16 ? Mi355xNative.KIND_BF16 : Mi355xNative.KIND_F32"
