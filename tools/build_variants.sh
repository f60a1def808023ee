#!/bin/bash
# Diagnostic builds of libfedcodec: ablations (FC_ABL bits), phase stamps, occupancy.
set -e
cd "$(dirname "$0")/.."
V="stamps=FC_STAMPS"
for v in ${ABL-1 2 4 8 15}; do V="$V abl$v=FC_ABL=$v"; done
for w in ${WAVES-4 6 8}; do V="$V w$w=FC_ENC_WAVES=$w"; done
python3 -m federated_amd.build $V
