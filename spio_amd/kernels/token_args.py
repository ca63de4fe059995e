"""Arguments of the kernels over sequences of tokens: the structures of csrc/spio_token_args.h, filled by field name.

The header is the one list of the fields, which the device code and the native call path include.
"""

import ctypes
import re
import struct
from functools import lru_cache
from typing import Tuple

from ..compiler.compile_kernel import read_source

HEADER = "spio_token_args.h"


@lru_cache(maxsize=None)
def fields_of(name: str) -> Tuple[Tuple[str, str], ...]:
    """(type, name) of the fields of a structure, in their order."""
    text = re.sub(r"//[^\n]*", "", read_source(HEADER))
    body = re.search(r"struct %s \{(.*?)\};" % name, text, re.DOTALL).group(1)
    out = []
    for declaration in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"((?:const )?(?:void|float|double|long long))\s*(.*)", declaration, re.DOTALL).groups()
        for field in (f.strip() for f in names.split(",")):
            out.append(("pointer" if field.startswith("*") else kind, field.lstrip("* ")))
    # "const float* a" has its star beside the type
    return tuple((k, f) for k, f in out)


class Arguments:
    """One filled structure; keeps the tensors it points into."""

    def __init__(self, name: str, **values):
        fields = fields_of(name)
        self.tensors = [v for v in values.values() if hasattr(v, "data_ptr")]
        slots = []
        for kind, field in fields:
            value = values.pop(field, None)
            if value is None:
                slots.append(0)
            elif hasattr(value, "data_ptr"):
                assert kind == "pointer", f"{field} is no tensor"
                slots.append(value.data_ptr())
            elif kind == "double":
                slots.append(struct.unpack("<Q", struct.pack("<d", float(value)))[0])
            else:
                assert kind == "long long", f"{field} is a tensor"
                slots.append(int(value) & 0xFFFFFFFFFFFFFFFF)
        assert not values, f"{name} has no fields {tuple(values)}"
        self.array = (ctypes.c_uint64 * len(slots))(*slots)
