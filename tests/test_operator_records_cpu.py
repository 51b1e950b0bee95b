"""The argument records of the ctypes binding against the header: a compiled program prints where the C compiler puts each field."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from ascend_kernel import _capi

ROOT = Path(__file__).resolve().parent.parent
KINDS = {"float": ctypes.c_float, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "uint32_t": ctypes.c_uint32}


def declared():
    """{record: [(field, type as ctypes has it)]} of the header, in order."""
    text = (ROOT / "include" / "ssd_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    records = {}
    for name, body in re.findall(r"typedef struct (Ssd\w+) \{(.*?)\} \1;", text, flags=re.S):
        fields = []
        for line in filter(None, (part.strip() for part in body.split(";"))):
            kind, names = re.match(r"((?:const )?\w+)\s*(.*)", line, flags=re.S).groups()
            kind = kind.replace("const ", "")
            for item in names.split(","):
                stars, field, count = re.fullmatch(r"\s*(\**)\s*(\w+)(?:\[(\d+)\])?\s*", item).groups()
                if stars:
                    of = ctypes.c_void_p
                else:
                    of = KINDS.get(kind) or getattr(_capi, kind)
                fields.append((field, of * int(count) if count else of))
        records[name] = fields
    return records


RECORDS = declared()


def test_every_record_is_mirrored():
    assert len(RECORDS) == 11 and all(hasattr(_capi, name) for name in RECORDS)


@pytest.mark.parametrize("name", RECORDS)
def test_fields_in_order(name):
    assert [(f, t) for f, t in getattr(_capi, name)._fields_] == RECORDS[name]


def test_places_and_sizes(tmp_path):
    lines = [f'printf("{name} %zu\\n", sizeof({name}));' for name in RECORDS]
    lines += [f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));' for name, fields in RECORDS.items() for field, _ in fields]
    source = tmp_path / "places.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ssd_b200.h"\nint main(void) {\n' + "\n".join(lines) +
                      "\nreturn 0;\n}\n")
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(source), "-o", str(tmp_path / "places")], check=True)
    places = subprocess.run([str(tmp_path / "places")], check=True, capture_output=True, text=True).stdout.split()
    places = dict(zip(places[::2], map(int, places[1::2])))
    for name, fields in RECORDS.items():
        record = getattr(_capi, name)
        assert ctypes.sizeof(record) == places[name], name
        for field, _ in fields:
            assert getattr(record, field).offset == places[f"{name}.{field}"], (name, field)
