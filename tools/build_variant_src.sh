#!/bin/bash
# Like build_variant.sh, but the unit is compiled from a given source file (an experiment kept out of
# the tree, e.g. under .dev/):   tools/build_variant_src.sh NAME UNIT SRC.hip "-DFLAGS..."
set -e
cd "$(dirname "$0")/.."
mkdir -p tools/variants
FLAGS=$(python3 -c "import __graft_entry__ as e; print(*e.FLAGS)")   # the in-tree build's
P=./-gan-_amd
U=$2
cp "$3" $P/csrc/.ab_src_$U.hip
/opt/rocm/bin/hipcc $FLAGS $4 -I$P/csrc -c $P/csrc/.ab_src_$U.hip -o tools/variants/$1.o
rm -f $P/csrc/.ab_src_$U.hip
OBJS=""
for u in $(python3 -c "import __graft_entry__ as e, os; print(*[os.path.basename(s)[:-4] for s in e.SOURCES])"); do
  [ "$u" = "$U" ] || OBJS="$OBJS $P/build/$u.hip.o"
done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -fPIC -shared -o tools/variants/$1.so tools/variants/$1.o $OBJS
rm tools/variants/$1.o
